"""B200-native Block Delta Memory (BDM) layer hot path.

Drop-in for the reference module's layer API (``BSDMConfig``,
``BlockSparseDeltaMemory(config, layer_id=, seed=)``, ``forward`` /
``prefill`` / ``step``; training backward; the ``BDMLanguageModel`` shell).  The bank path -- controllers epilogue, product-key
router, causal dispatch, per-bank recurrence, read combine, decode step -- runs
in hand-written sm_100a kernels behind the C ABI in ``include/bdm_b200.h``
(``libbdm_b200.so`` in this directory, built by ``python -m bdm_b200.build``).

Beside the bank memory: decay attention (``decay_attention``, ``decay_attention_step``, the
``DecayAttention`` mixer), language models that interleave the two (``HybridLanguageModel``), and beam
search over their states (``beam_select``, ``reorder_states``, ``beam_search``).
"""
from .beam import BeamStep, beam_search, beam_select, reorder_states
from .config import BDMConfig, BSDMConfig, near_square_factors, state_interval
from .decay import DecayAttention, decay_attention, decay_attention_step
from .hybrid import HybridLanguageModel
from .layer import BankedDeltaMemory, BlockSparseDeltaMemory, SharedResidualRouter
from .lm import BDMLanguageModel, LanguageModelConfig

__all__ = ['BDMConfig', 'BSDMConfig', 'BankedDeltaMemory', 'BlockSparseDeltaMemory', 'SharedResidualRouter',
           'BDMLanguageModel', 'LanguageModelConfig', 'near_square_factors', 'state_interval',
           'DecayAttention', 'HybridLanguageModel', 'decay_attention', 'decay_attention_step',
           'BeamStep', 'beam_search', 'beam_select', 'reorder_states']
