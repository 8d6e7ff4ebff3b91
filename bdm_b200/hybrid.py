"""Language model that interleaves bank memory layers with decay attention.

The same shell as ``BDMLanguageModel`` (embedding, blocks of mixer and feed-forward, head) with the mixers
of chosen layers replaced by ``DecayAttention``: the bank memory stores sparsely by content, the decay
heads carry the recent context densely.  Training, ``prefill``, ``step``, ``capture_step`` and
``beam_search`` work as on ``BDMLanguageModel``; the cache of a decay layer is its FP32 state.
"""
from __future__ import annotations

from .decay import DecayAttention
from .lm import BDMLanguageModel, LanguageModelConfig


class HybridLanguageModel(BDMLanguageModel):
    """``decay_layers``: indices of the layers whose mixer is decay attention (default: every second one)."""

    def __init__(self, config: LanguageModelConfig, *, decay_layers=None, decay_heads=None, decay_kv_heads=None,
                 backend: str = 'role'):
        super().__init__(config, backend=backend)
        layers = range(1, config.layers, 2) if decay_layers is None else decay_layers
        self.decay_layers = tuple(sorted(set(int(i) for i in layers)))
        if any(not 0 <= i < config.layers for i in self.decay_layers):
            raise ValueError('decay_layers must be indices of the model\'s layers')
        heads = config.memory.num_heads if decay_heads is None else decay_heads
        for i in self.decay_layers:
            self.layers[i].attention = DecayAttention(self.dim, heads, kv_heads=decay_kv_heads,
                                                      norm_eps=config.memory.norm_eps,
                                                      seed=config.seed * 100_000 + 9000 + i)
