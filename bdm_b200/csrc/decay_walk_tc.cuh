// Decay attention on the tensor cores: the walk of decay_walk.cuh for BF16 operands (kernel template; one
// translation unit per pair of tile widths instantiates it).
//
// One CTA walks the 64-token chunks of one segment of one (row, head).  Everything is computed transposed,
// so that the state's and the outputs' value columns are the lanes of tensor memory:
//   A    = Qa Kb^T                 [i, j]   operands as TMA leaves them (K-major)
//   P    = scale A * lam^(i-j), masked      -> BF16 in shared memory, [i][j]
//   O1^T = Vc^T P^T                [dv, i]  Vc read MN-major
//   O2^T = S^T Qa^T                [dv, i]  S^T is a BF16 operand in tensor memory
//   T^T  = V'^T Kb                 [dv, dk] V' = lam^. Vc as two or three BF16 terms in tensor memory, Kb MN-major
//   out  = O1 + scale lam^. O2,    S <- lam^n S + T
// The state itself stays in registers in FP32.  Roundings to BF16: P and the copy of S that is read (one
// rounding each, as large as the output's own).  V' is split into three terms (24 bits) where a state is
// returned: the state is then as near as an FP32 sum, over any number of chunks (65536 to 400000 tokens of one sign
// without decay: 1.5e-6 at the worst element).  Where none is, two terms (an error of 2^-17 beside the outputs' 2^-9)
// are enough.
//
// Roles (23 warps of 24): 0-7 carry the state (a quadrant's value columns, half of the key columns), 8-11 scale V',
// 12-15 the outputs, 16-19 P, 20 and 22 MMA, 21 TMA.  V' is made and T issued in two halves of 32 tokens, so that
// the scaling of one overlaps the product of the other (in the state launch by two groups, 8-11 and 12-15, at once).
// V' is in tensor memory because shared memory's bandwidth is what the products and copies share: as a
// shared-memory operand it took 768 more of its cycles per chunk.
// The roles' loops are kept short on purpose: five roles' unrolled code does not fit the instruction cache
// (2048 tokens x 148 heads of 128: 100 us unrolled, 78 us rolled, with one set of roles).
// Wider values than 64 take one CTA with 128 lanes, or, where rows are few, two with 64 columns each.
// The scores, and value widths up to 64, use M = 64 products, whose 64 rows are 16 lanes of each quadrant, so
// that all four schedulers share the work; wider values use all 128 lanes.
// Every wait is bounded; one that gives up sets the status word and lets the CTA drain.
// Values that are not finite: a masked score, exactly zero, still multiplies what it masks, so a token's infinity or
// NaN would reach the tokens before it.  The output warps look for NaN in what they write, which costs the walk at
// width 64 about 7 %, and sum such outputs again.
// Bound: HBM at 148 rows (4096 tokens x 148 heads of 128 in 109 to 117 us, 95 at the copy rate), a chunk's chain of
// hand-offs (1.7 us at 128 columns, 1.0 at 64) where there are fewer.
#pragma once

#include "decay_walk.cuh"
#include "tcgen05.cuh"

#include <cuda.h>

#include <mutex>

namespace bdm {
namespace walk {

constexpr int kTcThreads = 768;
// Registers: 6 groups of 4 warps, 80 per thread at launch (480 in all), dealt out as 2 x 112 (state) + 72 (V') + 80
// (outputs) + 64 (P) + 40 (loads and products).
constexpr int kLaunchRegs = 80;
constexpr int kStateRegs = 112, kScaleRegs = 72, kOutRegs = 80, kScoreRegs = 64, kMmaRegs = 40;
static_assert(2 * kStateRegs + kScaleRegs + kOutRegs + kScoreRegs + kMmaRegs <= 6 * kLaunchRegs, "register shares");
constexpr int kBox = 64 * 128;  // bytes of a TMA box: 64 tokens x 64 BF16 columns
constexpr int kStateWarps = 8, kScaleWarp = 8, kOutWarp = 12, kScoreWarp = 16, kMmaWarp = 20, kTmaWarp = 21,
              kOutMmaWarp = 22;
constexpr int kMaxStages = 8;
constexpr int kSmemMax = 227 * 1024;
constexpr long long kWaitCycles = 4000000000ll;  // about 2 s
constexpr unsigned long long kWaitNs = 2000000000ull;

// tensor memory columns
constexpr uint32_t kColA = 0, kColO1 = 64, kColO2 = 128, kColT = 192, kColS = 320, kColV = 384;
// State launch: the chunks whose products gather in one T before it is added to the FP32 state.  Tensor-core sums are
// cut off, not rounded, and a long one drifts: of 65536 tokens of one sign x 74 heads of 64, 3.4e-5 of the state was lost
// with whole sub-segments in one T, and 1e-8 is in groups of 4 (1.5e-6 at the worst element, as in FP32).  Two T's, so
// that one is read while the next group gathers (1 x 65536 x 8 x 128: 179 us, with one sum 177.5).
constexpr int kGroup = 4;
constexpr uint32_t kColT2 = 0;

struct Maps {
    CUtensorMap a, b, c, out;
};
struct TcParams {
    Params p;
    int amul[3], bmul[3];  // 0 where the operand's batch (head) is shared by all: a, b, c
    int sub, scps;         // state launch: sub-segments of a segment, chunks of one
    int longest_first;     // rows are dealt out by length
    int vsplit;            // CTAs that share a row's value columns, 64 each (1: one has them all)
    float *z;              // its states, [batch*heads, (nseg - 1) * sub, wc * wab]
};

// A parity tells a phase from the next only, so no waiter may fall two phases behind: each barrier's next phase
// needs something that its waiter gives after the wait (P's two buffers have one barrier each for that reason).
struct Bars {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t vready[2], tpart[2], tfree, sready;              // V' halves, T halves, T read, S written
    uint64_t tgroup[2], tdrained[2];                          // state launch: a group's T whole, read
    uint64_t adone, pready, pfree[2], odone, oissued[2], ofree;  // A, P, P read, O, O issued, O read
    uint64_t zeroed, ofull, oempty, drain[2];                 // row's end cleared, output buffers, issuers' last products
};

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Two FP32 values in one register pair, for the packed FP32 instructions.
struct F2 {
    unsigned long long v;
};
__device__ __forceinline__ F2 make2(float x, float y) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r.v) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 split2(F2 a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ uint32_t pack2(F2 a) {
    const float2 x = split2(a);
    return pack_bf16(x.x, x.y);
}
__device__ __forceinline__ float bf16_lo(uint32_t r) { return __uint_as_float(r << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t r) { return __uint_as_float(r & 0xffff0000u); }
__device__ __forceinline__ F2 unpack2(uint32_t r) { return make2(bf16_lo(r), bf16_hi(r)); }
// Two values as N = 2 or 3 BF16 terms each.
template <int N> __device__ __forceinline__ void terms(F2 x, uint32_t &hi, uint32_t &mid, uint32_t &lo) {
    const F2 minus = make2(-1.f, -1.f);
    hi = pack2(x);
    x = fma2(unpack2(hi), minus, x);
    mid = pack2(x);
    if constexpr (N == 3) {
        x = fma2(unpack2(mid), minus, x);
        lo = pack2(x);
    }
}

// Running maximum of BF16 pairs that keeps a NaN, and whether it has met one.
__device__ __forceinline__ uint32_t max_nan(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ bool met_nan(uint32_t a) {  // such a NaN is 0x7fff
    return ((a & 0x7fff7fffu) + 0x00010001u) & 0x80008000u;
}

__device__ __forceinline__ bool wait_slow(uint64_t *m, unsigned parity, volatile int *dead) {
    const long long t0 = clock64();
    for (int i = 0; i < (1 << 28); ++i) {
        if (tc::mbar_test_for(m, parity, 1000)) return true;
        if ((i & 15) == 15 && (*dead || clock64() - t0 > kWaitCycles)) break;
    }
    *dead = 1;
    return false;
}

// Stages of the load pipeline: what shared memory holds beside two buffers of P and of outputs.
template <int DKB, int VB, bool STATE_ONLY> constexpr int stages_of() {
    const int stage = (STATE_ONLY ? DKB + VB : 2 * DKB + VB) * kBox;
    const int n = (kSmemMax - 1024 - 3072 - 2 * (1 + VB) * kBox) / stage;
    return n > kMaxStages ? kMaxStages : n;
}

// DKB, VB: 64-column boxes of a / b and of c.  TERMS of V'.
template <int DKB, int VB, int TERMS, typename OT, bool STATE_ONLY>
__global__ void __launch_bounds__(kTcThreads, 1) decay_walk_tc_kernel(const TcParams tp, const __grid_constant__ Maps maps) {
    extern __shared__ char raw[];
    __shared__ Bars bar;
    __shared__ float pw[kChunk + 1];     // lam^m
    __shared__ float ow[2 * kChunk];     // scale lam^. of a full chunk's tokens reading the state
    __shared__ float vw[2 * kChunk];     // lam^. of a full chunk's tokens writing it
    __shared__ float wt[2 * kChunk];     // scale lam^d at kChunk + d, 0 for d < 0
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int dead;
    const Params &p = tp.p;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    char *smem = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    constexpr int kStage = (STATE_ONLY ? DKB + VB : 2 * DKB + VB) * kBox;
    constexpr int kOffB = STATE_ONLY ? 0 : DKB * kBox, kOffC = kOffB + DKB * kBox;
    constexpr int DK = DKB * 64, M = VB * 64;
    constexpr int kHalves = VB;  // 16-lane halves of a quadrant that hold value columns
    constexpr int stages = stages_of<DKB, VB, STATE_ONLY>();
    char *sP = smem + stages * kStage;

    int64_t id = blockIdx.x;
    const int voff = tp.vsplit > 1 ? (int)(id % tp.vsplit) * 64 : 0;  // neighbours read the same a and b
    id /= tp.vsplit;
    const int segs = STATE_ONLY ? (p.nseg - 1) * tp.sub : p.nseg;
    const int seg = (int)(id % segs);
    int64_t bh = id / segs;
    if (tp.longest_first) {
        // rows in the order of their lengths, so that the last wave of CTAs is short ones
        __shared__ int pick;
        const int want = (int)(bh / p.heads), i = threadIdx.x;
        if (i < p.batch) {
            const int64_t mine = row_tokens(p, i);
            int rank = 0;
            for (int j = 0; j < p.batch; ++j) {
                const int64_t other = row_tokens(p, j);
                rank += other > mine || (other == mine && j < i);
            }
            if (rank == want) pick = i;
        }
        __syncthreads();
        bh = (int64_t)pick * p.heads + bh % p.heads;
    }
    const int64_t b = bh / p.heads;
    const int h = (int)(bh % p.heads);
    const float g = head_log_decay(p, h);
    Span sp;
    if (STATE_ONLY) {  // the first (last) segment's state is not asked for in the forward (reverse) walk
        sp.n = row_tokens(p, b);
        sp.chunks = (sp.n + kChunk - 1) / kChunk;
        sp.c0 = (int64_t)(seg + (p.reverse ? tp.sub : 0)) * tp.scps;
        sp.c1 = sp.c0 + tp.scps;
        if (sp.c0 > sp.chunks) sp.c0 = sp.chunks;
        if (sp.c1 > sp.chunks) sp.c1 = sp.chunks;
    } else {
        sp = span_of(p, row_tokens(p, b), seg);
    }
    const int steps = (int)(sp.c1 - sp.c0);

    if (threadIdx.x <= kChunk) pw[threadIdx.x] = threadIdx.x ? expf(g * (float)threadIdx.x) : 1.f;
    if (threadIdx.x < 2 * kChunk) {
        // a chunk with fewer tokens starts later in the tables that count down
        const int i = threadIdx.x;
        auto lam = [&](int e) { return e < 0 || e > kChunk ? 0.f : (e ? expf(g * (float)e) : 1.f); };
        ow[i] = p.scale * lam(p.reverse ? kChunk - 1 - i : i + 1);
        vw[i] = lam(p.reverse ? i + 1 : kChunk - 1 - i);
        wt[i] = p.scale * lam(i - kChunk);
    }
    if (threadIdx.x == 0) {
        dead = 0;
        for (int i = 0; i < stages; ++i) {
            tc::mbar_init(&bar.full[i], 1);
            tc::mbar_init(&bar.empty[i], STATE_ONLY ? 1 : 2);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&bar.vready[i], 4);
            tc::mbar_init(&bar.tpart[i], 1);
            tc::mbar_init(&bar.tgroup[i], 1);
            tc::mbar_init(&bar.tdrained[i], kStateWarps);
            tc::mbar_init(&bar.pfree[i], 1);
            tc::mbar_init(&bar.oissued[i], 1);
        }
        tc::mbar_init(&bar.tfree, kStateWarps);
        tc::mbar_init(&bar.sready, kStateWarps);
        tc::mbar_init(&bar.adone, 1);
        tc::mbar_init(&bar.pready, 4);
        tc::mbar_init(&bar.odone, 1);
        tc::mbar_init(&bar.ofree, 4);
        tc::mbar_init(&bar.zeroed, 4);
        tc::mbar_init(&bar.ofull, 4);
        tc::mbar_init(&bar.oempty, 1);
        tc::mbar_init(&bar.drain[0], 1);
        tc::mbar_init(&bar.drain[1], 1);
        tc::mbar_fence_init();
    }
    if (warp == kMmaWarp) tc::tmem_alloc(&tmem_slot, 512);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const uint32_t tmem = tmem_slot;

    // bounded waits, the second for a whole warp with one answer for its lanes; false once any has given up
    auto wait = [&](uint64_t *m, unsigned parity) -> bool { return tc::mbar_test(m, parity) || wait_slow(m, parity, &dead); };
    auto wait_warp = [&](uint64_t *m, unsigned parity) -> bool { return __all_sync(0xffffffffu, wait(m, parity)); };
    // this warp's tensor-memory accesses (loads too) are done before whoever waits on m goes on
    auto arrive = [&](uint64_t *m) {
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(m);
    };
    // first token and valid tokens of the n-th chunk of the walk
    const int tokens = (int)sp.n, time = (int)p.time;
    const int first = (int)(p.reverse ? sp.c1 - 1 : sp.c0) * kChunk, stride = p.reverse ? -kChunk : kChunk;
    auto start_of = [&](int n) -> int { return first + n * stride; };
    auto valid_of = [&](int n) -> int { return min(tokens - start_of(n), kChunk); };
    const int quad = warp & 3;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    constexpr int kQuadCols = 16 * kHalves;  // value columns of a quadrant

    // V' of the half chunks half0, half0 + every, ... (32 tokens each), by the four warps of a group
    auto scale_values = [&](int half0, int every, int ctid) -> bool {
        // this lane's row of the matrices it loads: two of 8 tokens by two of 8 columns
        const int mrow = ((lane >> 4) * 8 + (lane & 7)) * 128, mcol = (lane >> 3) & 1;
        int st = 0, phase = 0;  // stage of the chunk, parity of its barrier
        for (int hs = half0; hs < 2 * steps; hs += every) {
            const int n = hs >> 1, hb = hs & 1;
            const int valid = valid_of(n);
            if (hb == 0 || every == 2) {
                if (!wait_warp(&bar.full[st], phase)) return false;
                if (valid < kChunk && start_of(n) + valid < time) {
                    // tokens past the row's length may hold anything: zero them for the products over j
                    if (hb == 0) {
                        uint4 *kb = reinterpret_cast<uint4 *>(smem + st * kStage + kOffB);
#pragma unroll 1
                        for (int i = ctid; i < (DKB + VB) * kBox / 16; i += 128)
                            if ((i % (kBox / 16)) / 8 >= valid) kb[i] = make_uint4(0, 0, 0, 0);
                        tc::fence_async_smem();
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(&bar.zeroed);  // once at most: a row has one such chunk
                    }
                    if (!wait_warp(&bar.zeroed, 0)) return false;
                }
            }
            if (n > 0) {
                if (!wait_warp(&bar.tpart[hb], (n - 1) & 1)) return false;
                tc::fence_after_sync();
            }
            // in the state launch chunks are added up without a carry: their distance to the segment's end counts too
            float far = 1.f;
            if (STATE_ONLY) {
                const int64_t last = sp.c1 * kChunk < sp.n ? sp.c1 * kChunk : sp.n;
                const int64_t gap = p.reverse ? start_of(n) - sp.c0 * kChunk : last - start_of(n) - valid;
                far = gap ? expf(g * (float)gap) : 1.f;
            }
            // 16 tokens by this quadrant's columns at a time: transposed on the way in, scaled, and split into BF16
            // terms as the fragments that tensor memory takes
            const float *w = vw + (p.reverse ? 0 : kChunk - valid) + hb * 32 + 2 * (lane & 3);
            const char *src = smem + st * kStage + kOffC + (VB == 2 ? (quad >> 1) * kBox : 0) + hb * 32 * 128 + mrow;
            const int c0 = VB == 2 ? (quad & 1) * 4 : quad * 2;
#pragma unroll (VB == 1 ? 2 : 1)
            for (int q = 0; q < 2; ++q, src += 16 * 128, w += 16) {
                const F2 w0 = make2(w[0] * far, w[1] * far), w1 = make2(w[8] * far, w[9] * far);
                uint32_t r[kHalves][4];
#pragma unroll
                for (int d = 0; d < kHalves; ++d)
                    tc::ldmatrix_x4_trans(src + (((c0 + d * 2 + mcol) ^ (lane & 7)) << 4), r[d]);
#pragma unroll
                for (int d = 0; d < kHalves; ++d) {
                    uint32_t t[3][4];
#pragma unroll
                    for (int m = 0; m < 4; ++m) terms<TERMS>(mul2(m < 2 ? w0 : w1, unpack2(r[d][m])), t[0][m], t[1][m], t[2][m]);
#pragma unroll
                    for (int u = 0; u < TERMS; ++u) {
                        const uint32_t at = tmem + lanes + kColV + hb * 48 + u * 16 + q * 8;
                        tc::tmem_st_16x128b_x2(at + (d << 20), t[u][0], t[u][1], t[u][2], t[u][3]);
                    }
                }
            }
            if ((hb || every == 2) && ++st == stages) st = 0, phase ^= 1;
            tc::tmem_wait_st();
            arrive(&bar.vready[hb]);
        }
        return true;
    };

    if (warp < kStateWarps) {
        tc::regs_up<kStateRegs>();
        // ------------------------------------------------------------------ state
        // Fragments: S[d][4 b + 2 r + e] is key column k0 + 8 b + 2 (lane % 4) + e of value column
        // quad * kQuadCols + 16 d + 8 r + lane / 4.
        constexpr int KC = DK / 2;
        const int k0 = (warp >> 2) * KC, kl = k0 + 2 * (lane & 3), v0 = voff + quad * kQuadCols + (lane >> 2);
        const int64_t size = (int64_t)p.wab * p.wc;
        F2 S[kHalves][KC / 4];
#pragma unroll
        for (int d = 0; d < kHalves; ++d)
#pragma unroll
            for (int i = 0; i < KC / 4; ++i) S[d][i] = make2(0.f, 0.f);
        if constexpr (!STATE_ONLY) {
            const bool before = p.nseg > 1 && (p.reverse ? seg < p.nseg - 1 : seg > 0);
            const float *zs = p.seg + (bh * p.nseg + seg) * size;
            if (p.nseg > 1) asm volatile("griddepcontrol.wait;\n" ::: "memory");
            const int64_t end = sp.c1 * kChunk < sp.n ? sp.c1 * kChunk : sp.n;
            const int64_t far = p.reverse ? sp.n - end : sp.c0 * kChunk;
            const float w = p.state_in ? (far ? expf(g * (float)far) : 1.f) * p.in_mul : 0.f;
            const float *x = p.state_in ? p.state_in + bh * size : nullptr;
            // every load at an address that exists, the ones outside selected away: no branch holds the next one up
            auto gather = [&](const float *from, bool transposed, float mul) {
#pragma unroll
                for (int d = 0; d < kHalves; ++d)
#pragma unroll
                    for (int i = 0; i < KC / 4; ++i) {
                        const int v = v0 + 16 * d + 8 * (i & 1), k = kl + 8 * (i >> 1);
                        float s[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const bool in = v < p.wc && k + e < p.wab;
                            const int at = transposed ? v * p.wab + k + e : (k + e) * p.wc + v;
                            const float f = __ldg(from + (in ? at : 0));
                            s[e] = in ? f : 0.f;
                        }
                        S[d][i] = fma2(make2(mul, mul), make2(s[0], s[1]), S[d][i]);
                    }
            };
            if (before) gather(zs, true, 1.f);
            if (p.state_in) gather(x, p.in_t, w);
        }
        auto add_products = [&](uint32_t col, F2 carry) {
#pragma unroll
            for (int d = 0; d < kHalves; ++d)
#pragma unroll
                for (int i = 0; i < KC; i += 32) {
                    float t[16];
                    tc::tmem_ld_16x256b_x4(tmem + lanes + (d << 20) + col + k0 + i, t);
                    tc::tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 8; ++e) S[d][i / 4 + e] = fma2(carry, S[d][i / 4 + e], make2(t[2 * e], t[2 * e + 1]));
                }
        };
        bool ok = true;
        if constexpr (STATE_ONLY)
            for (int i = 0; ok && i * kGroup < steps; ++i) {
                ok = wait_warp(&bar.tgroup[i & 1], (i >> 1) & 1);
                if (!ok) break;
                tc::fence_after_sync();
                add_products(i & 1 ? kColT2 : kColT, make2(1.f, 1.f));
                arrive(&bar.tdrained[i & 1]);
            }
        for (int n = 0; !STATE_ONLY && ok && n <= steps; ++n) {
            if (n > 0) {
                ok = wait_warp(&bar.tpart[1], (n - 1) & 1);
                if (!ok) break;
                tc::fence_after_sync();
                const float f = pw[valid_of(n - 1)];
                add_products(kColT, make2(f, f));
                if (n == steps) break;
                arrive(&bar.tfree);
                ok = wait_warp(&bar.odone, (n - 1) & 1);  // the last chunk's reads of S are over
                if (!ok) break;
                tc::fence_after_sync();
            }
            if (n < steps) {
#pragma unroll
                for (int d = 0; d < kHalves; ++d)
#pragma unroll
                    for (int i = 0; i < KC / 4; i += 4)
                        tc::tmem_st_16x128b_x2(tmem + lanes + (d << 20) + kColS + k0 / 2 + i * 2, pack2(S[d][i]), pack2(S[d][i + 1]),
                                               pack2(S[d][i + 2]), pack2(S[d][i + 3]));
                tc::tmem_wait_st();
                arrive(&bar.sready);
            }
        }
        if (ok && (STATE_ONLY || (p.state_out && sp.last))) {
            float *z = STATE_ONLY ? tp.z + (bh * segs + seg) * size : p.state_out + bh * size;
            const float mul = STATE_ONLY ? 1.f : p.out_mul;
            const bool t = STATE_ONLY || p.out_t;
#pragma unroll
            for (int d = 0; d < kHalves; ++d)
#pragma unroll
                for (int i = 0; i < KC / 4; ++i) {
                    const int v = v0 + 16 * d + 8 * (i & 1), k = kl + 8 * (i >> 1);
                    const float2 s = split2(S[d][i]);
                    if (v >= p.wc) continue;
                    if (k < p.wab) z[t ? (int64_t)v * p.wab + k : (int64_t)k * p.wc + v] = s.x * mul;
                    if (k + 1 < p.wab) z[t ? (int64_t)v * p.wab + k + 1 : (int64_t)(k + 1) * p.wc + v] = s.y * mul;
                }
        }
    } else if (warp < kOutWarp) {
        tc::regs_down<kScaleRegs>();
        scale_values(0, STATE_ONLY ? 2 : 1, threadIdx.x - kScaleWarp * 32);
    } else if (warp < kScoreWarp) {
        // ---------------------------------------------------------------- outputs
        if constexpr (!STATE_ONLY) {
            OT *out = static_cast<OT *>(p.out) + b * p.os[0] + h * p.os[2];
            constexpr bool kTma = sizeof(OT) == 2;  // BF16 outputs leave by TMA, FP32 ones (partial sums) by plain stores
            const int mtok = ((lane >> 4) * 8 + (lane & 7)) * 128, mcol = (lane >> 3) & 1;
            const int c0 = VB == 2 ? (quad & 1) * 4 : quad * 2;
            for (int n = 0; n < steps; ++n) {
                const int t0 = start_of(n), valid = valid_of(n);
                char *stage = sP + (2 + (n & 1) * VB) * kBox;  // BF16 outputs on their way, [token][column]: the map's boxes
                if (kTma && n > 1) {
                    if (warp == kOutWarp && lane == 0) {
                        tc::tma_store_wait_read<1>();
                        tc::mbar_arrive(&bar.oempty);
                    }
                    if (!wait_warp(&bar.oempty, n & 1)) break;
                }
                if (!wait_warp(&bar.odone, n & 1)) break;
                tc::fence_after_sync();
                const float *w0 = ow + (p.reverse ? kChunk - valid : 0) + 2 * (lane & 3);
                uint32_t seen = 0;
                // 16 columns by 32 tokens at a time.  Fragments: this lane has tokens 8 b + 2 (lane % 4) + {0, 1} of
                // column 16 d + lane / 4 (+ 8).
#pragma unroll 1
                for (int q = 0; q < 2 * kHalves; ++q) {
                    const int d = q >> 1, i = q & 1;
                    float y[16], z[16];
                    const uint32_t at = tmem + lanes + (d << 20) + i * 32;
                    tc::tmem_ld_16x256b_x4(at + kColO2, y);
                    tc::tmem_ld_16x256b_x4(at + kColO1, z);
                    const float *w = w0 + i * 32;
                    F2 wo[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) wo[e] = make2(w[8 * e], w[8 * e + 1]);
                    tc::tmem_wait_ld();
                    F2 x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        x[e] = fma2(wo[e / 2], make2(y[2 * e], y[2 * e + 1]), make2(z[2 * e], z[2 * e + 1]));
                    const int r0 = i * 32 + 2 * (lane & 3);
                    if constexpr (kTma) {
                        uint32_t v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = pack2(x[e]);
                        if (valid < kChunk)  // padding gives zeros
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const int r = r0 + e / 2 * 8;
                                v[e] &= (r < valid ? 0xffffu : 0u) | (r + 1 < valid ? 0xffff0000u : 0u);
                            }
#pragma unroll
                        for (int e = 0; e < 8; ++e) seen = max_nan(seen, v[e]);
                        char *dst = stage + (VB == 2 ? (quad >> 1) * kBox : 0) + i * 32 * 128 + mtok +
                                    (((c0 + d * 2 + mcol) ^ (lane & 7)) << 4);
                        tc::stmatrix_x4_trans(dst, v[0], v[1], v[2], v[3]);
                        tc::stmatrix_x4_trans(dst + 16 * 128, v[4], v[5], v[6], v[7]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int r = r0 + e / 2 * 8, c = voff + quad * kQuadCols + d * 16 + (e & 1) * 8 + (lane >> 2);
                            float2 v = split2(x[e]);
                            v.x = r < valid ? v.x : 0.f;
                            v.y = r + 1 < valid ? v.y : 0.f;
                            seen = max_nan(seen, pack_bf16(v.x, v.y));
                            OT *o = out + (int64_t)(t0 + r) * p.os[1] + c;
                            if (c < p.wc && t0 + r < time) o[0] = v.x;
                            if (c < p.wc && t0 + r + 1 < time) o[p.os[1]] = v.y;
                        }
                    }
                }
                if (__builtin_expect(__any_sync(0xffffffffu, met_nan(seen)), 0)) {
                    // A masked score of zero times a value that is not finite, or a zero weight times such a score, is
                    // NaN.  The outputs that hold one although what they read of the state is finite are summed again,
                    // over the tokens that reach them only: a lane has a column.  Slow (up to 1 ms a chunk), but a chunk
                    // where this happens turns columns or rows of the state bad, which then need it no more.
                    __syncwarp();
                    const bf16 *pa = static_cast<const bf16 *>(p.a) + b * p.as[0] + (h / p.ag) * p.as[2] + t0 * p.as[1];
                    const bf16 *pb = static_cast<const bf16 *>(p.b) + b * p.bs[0] + (h / p.bg) * p.bs[2] + t0 * p.bs[1];
                    const bf16 *pc = static_cast<const bf16 *>(p.c) + b * p.cs[0] + (h / p.cg) * p.cs[2] + t0 * p.cs[1];
                    const int c = quad * kQuadCols + lane;
                    const bool mine = lane < kQuadCols && voff + c < p.wc;
#pragma unroll 1
                    for (int i = 0; i < valid; ++i) {
                        const float y = tc::tmem_ld1(tmem + lanes + kColO2 + i), z = tc::tmem_ld1(tmem + lanes + kColO1 + i);
                        tc::tmem_wait_ld();
                        const float read = ow[(p.reverse ? kChunk - valid : 0) + i] * y, sum = read + z;
                        const bool redo = mine && sum != sum && read == read;
                        if (!__any_sync(0xffffffffu, redo)) continue;
                        const int j0 = p.reverse ? i : 0, j1 = p.reverse ? valid : i + 1;
                        float o = read;
#pragma unroll 1
                        for (int j = j0; j < j1; ++j) {
                            float s = 0.f;
#pragma unroll 1
                            for (int k = lane; k < p.wab; k += 32)
                                s = fmaf(__bfloat162float(pa[i * p.as[1] + k]), __bfloat162float(pb[j * p.bs[1] + k]), s);
                            s = warp_sum(s) * wt[kChunk + (p.reverse ? j - i : i - j)];
                            if (mine) o = fmaf(__bfloat162float(__float2bfloat16_rn(s)), __bfloat162float(pc[j * p.cs[1] + voff + c]), o);
                        }
                        if (redo) {
                            if constexpr (kTma)
                                *reinterpret_cast<bf16 *>(stage + c / 64 * kBox + i * 128 + (((c & 63) >> 3 ^ (i & 7)) << 4) +
                                                          (c & 7) * 2) = __float2bfloat16_rn(o);
                            else
                                out[(int64_t)(t0 + i) * p.os[1] + voff + c] = o;
                        }
                        __syncwarp();
                    }
                }
                if (kTma) tc::fence_async_smem();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    tc::mbar_arrive(&bar.ofree);
                    if (kTma) tc::mbar_arrive(&bar.ofull);
                }
                if (kTma && warp == kOutWarp) {
                    if (!wait_warp(&bar.ofull, n & 1)) break;
                    if (lane == 0) {
#pragma unroll
                        for (int i = 0; i < VB; ++i) tc::tma_store_4d(&maps.out, stage + i * kBox, voff + i * 64, t0, h, (int)b);
                        tc::tma_store_commit();
                    }
                }
            }
            if (kTma && warp == kOutWarp && lane == 0) tc::tma_store_wait();
        } else {
            scale_values(1, 2, threadIdx.x - kOutWarp * 32);  // the halves that the other group leaves out
        }
    } else if (warp < kMmaWarp) {
        tc::regs_down<kScoreRegs>();
        // ------------------------------------------------------------ decayed scores P
        if constexpr (!STATE_ONLY) {
            // fragments: rows quad * 16 + lane / 4 (+ 8), columns 8 b + 2 (lane % 4) + {0, 1}
            const int row = quad * 16 + (lane >> 2), col = 2 * (lane & 3), step = p.reverse ? 1 : -1;
            const float *w0 = wt + kChunk + (p.reverse ? col - row : row - col);
            const int srow = quad * 16 + (lane & 15), scol = lane >> 4;  // stmatrix: this lane's row and block of 8 columns
            for (int n = 0; n < steps; ++n) {
                const int valid = valid_of(n);
                if (!wait_warp(&bar.adone, n & 1)) break;
                tc::fence_after_sync();
                if (n > 1 && !wait_warp(&bar.pfree[n & 1], ((n >> 1) - 1) & 1)) break;  // this buffer's last reads are over
                char *dst = sP + (n & 1) * kBox + srow * 128;
#pragma unroll 1
                for (int i = 0; i < 64; i += 32) {
                    float x[16];
                    tc::tmem_ld_16x256b_x4(tmem + lanes + kColA + i, x);
                    F2 w[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float *f = w0 + step * (i + e / 2 * 8 - (e & 1) * 8);  // row + 8 is 8 columns back
                        w[e] = make2(f[0], f[step]);
                    }
                    tc::tmem_wait_ld();
                    uint32_t r[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) r[e] = pack2(mul2(w[e], make2(x[2 * e], x[2 * e + 1])));
                    if (valid < kChunk)  // scores of tokens past the row's length may be anything
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int j = i + e / 2 * 8 + col;
                            r[e] &= (j < valid ? 0xffffu : 0u) | (j + 1 < valid ? 0xffff0000u : 0u);
                        }
#pragma unroll
                    for (int e = 0; e < 8; e += 4)
                        tc::stmatrix_x4(dst + (((i / 8 + e / 2 + scol) ^ (srow & 7)) << 4), r[e], r[e + 1], r[e + 2], r[e + 3]);
                }
                tc::fence_async_smem();
                arrive(&bar.pready);
            }
        }
    } else {
        tc::regs_down<kMmaRegs>();
        // Two issuers, one for the state's products and one for the outputs': a product costs its thread some 40
        // cycles and a wait 50 and more, and with one thread that chain was longer than the products.
        if (warp == kMmaWarp && tc::elect_one()) {
            // ------------------------------------------------------- products for the state
            constexpr uint32_t idT = tc::idesc_bf16(M, DK) | tc::kIdescMnB;
            uint32_t tile = tc::smem_u32(smem) + kOffB;
            bool ok = true;
            int st = 0;
            for (int n = 0; n < steps && ok; ++n) {
                uint64_t kb = tc::smem_desc_sw128_mn(tile, kBox);
                uint32_t va = tmem + kColV;
                uint32_t to = tmem + kColT;
                if (STATE_ONLY) {
                    const int i = n / kGroup;
                    to = tmem + (i & 1 ? kColT2 : kColT);
                    if (n % kGroup == 0 && i > 1 && !(ok = wait(&bar.tdrained[i & 1], ((i >> 1) - 1) & 1))) break;
                } else if (n > 0) {
                    if (!(ok = wait(&bar.tfree, (n - 1) & 1))) break;
                    // long products (N = 128) must not get ahead of the outputs', which more is waiting for
                    if (DKB == 2 && !(ok = wait(&bar.oissued[(n - 1) & 1], ((n - 1) >> 1) & 1))) break;
                }
#pragma unroll 1
                for (int hb = 0; hb < 2; ++hb, kb += 2 * 2048 / 16, va += 48) {
                    if (!(ok = wait(&bar.vready[hb], n & 1))) break;
                    tc::fence_after_sync();
#pragma unroll
                    for (int t = 0; t < TERMS; ++t)
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            tc::mma_bf16_tmem_a(to, va + t * 16 + k * 8, kb + k * 2048 / 16, idT,
                                                hb + t + k + (STATE_ONLY ? n % kGroup : 0) > 0);
                    tc::mma_commit(&bar.tpart[hb]);
                }
                if (STATE_ONLY && ok && (n % kGroup == kGroup - 1 || n + 1 == steps)) tc::mma_commit(&bar.tgroup[n / kGroup & 1]);
                tc::mma_commit(&bar.empty[st]);
                tile += kStage;
                if (++st == stages) st = 0, tile -= stages * kStage;
            }
            // no product may be in flight when the CTA ends, whatever happened to its consumers
            tc::mma_commit(&bar.drain[0]);
            tc::mbar_wait(&bar.drain[0], 0, kWaitNs);
        } else if (!STATE_ONLY && warp == kOutMmaWarp && tc::elect_one()) {
            // ----------------------------------------------------- products for the outputs
            constexpr uint32_t idQK = tc::idesc_bf16(64, 64);
            constexpr uint32_t idO1 = tc::idesc_bf16(M, 64) | tc::kIdescMnA;
            constexpr uint32_t idO2 = tc::idesc_bf16(M, 64);
            // descriptors of the buffers' starts; an offset adds its bytes / 16 to the low word
            const uint32_t base = tc::smem_u32(smem);
            const uint64_t dP = tc::smem_desc_sw128(tc::smem_u32(sP));
            auto scores = [&](int st) {
                uint64_t qa = tc::smem_desc_sw128(base + st * kStage), kb = qa + kOffB / 16;
#pragma unroll 1
                for (int i = 0; i < DKB; ++i, qa += kBox / 16, kb += kBox / 16)
#pragma unroll
                    for (int k = 0; k < 4; ++k) tc::mma_bf16(tmem + kColA, qa + k * 2, kb + k * 2, idQK, i + k > 0);
                tc::mma_commit(&bar.adone);
            };
            int st = 0, phase = 0;
            if (steps > 0 && wait(&bar.full[0], 0)) scores(0);
            for (int n = 0; n < steps; ++n) {
                const uint32_t tile = base + st * kStage;
                const int st1 = st + 1 == stages ? 0 : st + 1, phase1 = st + 1 == stages ? phase ^ 1 : phase;
                // P(n) is ready, so A is free: the next scores go first, P(n + 1) is what takes longest
                if (!wait(&bar.pready, n & 1)) break;
                tc::fence_after_sync();
                if (n + 1 < steps) {
                    if (!wait(&bar.full[st1], phase1)) break;
                    scores(st1);
                }
                if (!wait(&bar.sready, n & 1)) break;
                if (n > 0 && !wait(&bar.ofree, (n - 1) & 1)) break;
                const int valid = valid_of(n);
                if (valid < kChunk && start_of(n) + valid < time && !wait(&bar.zeroed, 0)) break;  // c past the row's end
                tc::fence_after_sync();
                uint64_t qa = tc::smem_desc_sw128(tile);
                uint32_t sa = tmem + kColS;
#pragma unroll 1
                for (int i = 0; i < DKB; ++i, qa += kBox / 16, sa += 32)
#pragma unroll
                    for (int k = 0; k < 4; ++k) tc::mma_bf16_tmem_a(tmem + kColO2, sa + k * 8, qa + k * 2, idO2, i + k > 0);
                const uint64_t vc = tc::smem_desc_sw128_mn(tile + kOffC, kBox), pn = dP + (n & 1) * kBox / 16;
#pragma unroll
                for (int k = 0; k < 4; ++k) tc::mma_bf16(tmem + kColO1, vc + k * 2048 / 16, pn + k * 2, idO1, k > 0);
                tc::mbar_arrive(&bar.oissued[n & 1]);
                tc::mma_commit(&bar.odone);
                tc::mma_commit(&bar.pfree[n & 1]);
                tc::mma_commit(&bar.empty[st]);
                st = st1, phase = phase1;
            }
            tc::mma_commit(&bar.drain[1]);
            tc::mbar_wait(&bar.drain[1], 0, kWaitNs);
        } else if (warp == kTmaWarp && tc::elect_one()) {
            // --------------------------------------------------------------- loads
            const int ha = (h / p.ag) * tp.bmul[0], hk = (h / p.bg) * tp.bmul[1], hc = (h / p.cg) * tp.bmul[2];
            const int ba = (int)b * tp.amul[0], bb = (int)b * tp.amul[1], bc = (int)b * tp.amul[2];
            int issued = 0, st = 0, phase = 0;
            for (int n = 0; n < steps; ++n) {
                if (n >= stages && !wait(&bar.empty[st], phase ^ 1)) break;
                char *dst = smem + st * kStage;
                const int t0 = start_of(n);
                tc::mbar_arrive_expect_tx(&bar.full[st], kStage);
#pragma unroll
                for (int i = 0; i < DKB; ++i) {
                    if (!STATE_ONLY) tc::tma_load_4d(dst + i * kBox, &maps.a, i * 64, t0, ha, ba, &bar.full[st]);
                    tc::tma_load_4d(dst + kOffB + i * kBox, &maps.b, i * 64, t0, hk, bb, &bar.full[st]);
                }
#pragma unroll
                for (int i = 0; i < VB; ++i) tc::tma_load_4d(dst + kOffC + i * kBox, &maps.c, voff + i * 64, t0, hc, bc, &bar.full[st]);
                issued = n + 1;
                if (++st == stages) st = 0, phase ^= 1;
            }
            // nor a copy
            for (int n = issued > stages ? issued - stages : 0; n < issued; ++n)
                tc::mbar_wait(&bar.full[n % stages], (n / stages) & 1, kWaitNs);
        }
    }
    __syncwarp();
    tc::fence_before_sync();
    __syncthreads();
    if constexpr (!STATE_ONLY) {
        // whole chunks past the row's length
        int64_t z0 = sp.chunks * kChunk, z1 = p.time;
        const int64_t s0 = (int64_t)seg * p.cps * kChunk, s1 = s0 + (int64_t)p.cps * kChunk;
        if (z0 < s0) z0 = s0;
        if (z1 > s1) z1 = s1;
        OT *out = static_cast<OT *>(p.out) + b * p.os[0] + h * p.os[2] + voff;
        constexpr int kLane = sizeof(OT) == 2 ? 8 : 1;  // BF16 rows are whole 16-byte units (TMA writes them too)
        const int cols = tp.vsplit > 1 ? min(p.wc - voff, 64) : p.wc, units = cols / kLane, per = kTcThreads / units;
        const int row = threadIdx.x / units, unit = threadIdx.x % units;
        if (row < per)
            for (int64_t t = z0 + row; t < z1; t += per) {
                if constexpr (sizeof(OT) == 2)
                    *reinterpret_cast<uint4 *>(out + t * p.os[1] + unit * 8) = make_uint4(0, 0, 0, 0);
                else
                    out[t * p.os[1] + unit] = 0.f;
            }
    }
    // A walk that overlaps the one before it does not end before that one has: what follows in the stream waits for
    // this walk only.
    if (!STATE_ONLY) asm volatile("griddepcontrol.wait;\n" ::: "memory");
    if (threadIdx.x == 0 && dead && p.status) *(volatile int *)p.status = 0x4;
    if (warp == kMmaWarp) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, 512);
    }
}

// One launch; `dependent`: its start may overlap the end of the launch before it (programmatic dependence).
template <int DKB, int VB, int TERMS, typename OT, bool STATE_ONLY>
int tc_launch(const TcParams &tp, const Maps &maps, bool dependent, cudaStream_t st) {
    constexpr int smem = stages_of<DKB, VB, STATE_ONLY>() * (STATE_ONLY ? DKB + VB : 2 * DKB + VB) * kBox +
                         2 * (1 + VB) * kBox + 1024;
    auto kernel = decay_walk_tc_kernel<DKB, VB, TERMS, OT, STATE_ONLY>;
    constexpr int kMaxDevices = 64;
    static std::mutex mu;
    static bool set[kMaxDevices];
    int dev = 0;
    if (int rc = cuda_status(cudaGetDevice(&dev))) return rc;
    if (dev < 0 || dev >= kMaxDevices) return BDM_ERR_UNSUPPORTED;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (!set[dev]) {
            if (int rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem))) return rc;
            // the state warps wait for the registers that the others give up: never launch with fewer than are dealt out
            cudaFuncAttributes fa;
            if (int rc = cuda_status(cudaFuncGetAttributes(&fa, kernel))) return rc;
            if (fa.numRegs < kLaunchRegs) return BDM_ERR_UNSUPPORTED;
            set[dev] = true;
        }
    }
    const int64_t blocks = tp.p.batch * tp.p.heads * tp.vsplit * (STATE_ONLY ? (int64_t)(tp.p.nseg - 1) * tp.sub : (int64_t)tp.p.nseg);
    if (blocks > 0x7fffffff) return BDM_ERR_UNSUPPORTED;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kTcThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = dependent ? 1 : 0;
    if (int rc = cuda_status(cudaLaunchKernelEx(&cfg, kernel, tp, maps))) return rc;
    return launch_status();
}

enum TcKind { kTcState, kTcBf16, kTcFloat };

// The launches of one pair of tile widths: terms 2 or 3.
template <int DKB, int VB> int tc_launch_any(const TcParams &tp, const Maps &maps, TcKind kind, int terms, bool dependent,
                                             cudaStream_t st) {
    if (kind == kTcState)
        return terms == 3 ? tc_launch<DKB, VB, 3, bf16, true>(tp, maps, dependent, st)
                          : tc_launch<DKB, VB, 2, bf16, true>(tp, maps, dependent, st);
    if (kind == kTcBf16)
        return terms == 3 ? tc_launch<DKB, VB, 3, bf16, false>(tp, maps, dependent, st)
                          : tc_launch<DKB, VB, 2, bf16, false>(tp, maps, dependent, st);
    return terms == 3 ? tc_launch<DKB, VB, 3, float, false>(tp, maps, dependent, st)
                      : tc_launch<DKB, VB, 2, float, false>(tp, maps, dependent, st);
}

#define BDM_TC_DECLARE(DKB, VB)                                                                                     \
    int tc_launch_##DKB##VB(const TcParams &tp, const Maps &maps, TcKind kind, int terms, bool dependent, cudaStream_t st)
BDM_TC_DECLARE(1, 1);
BDM_TC_DECLARE(1, 2);
BDM_TC_DECLARE(2, 1);
BDM_TC_DECLARE(2, 2);
#define BDM_TC_DEFINE(DKB, VB)                                                                                      \
    BDM_TC_DECLARE(DKB, VB) { return tc_launch_any<DKB, VB>(tp, maps, kind, terms, dependent, st); }

}  // namespace walk
}  // namespace bdm
