// Decay attention on the tensor cores: the walk of decay_walk.cuh for BF16 operands.
//
// One CTA walks the 64-token chunks of one segment of one (row, head).  Everything is computed transposed,
// so that the state's and the outputs' value columns are the 128 lanes of tensor memory and every product
// has M = 128:
//   A    = Qa Kb^T                 [i, j]   operands as TMA leaves them (K-major)
//   P    = scale A * lam^(i-j), masked      -> BF16 in shared memory, [i][j]
//   O1^T = Vc^T P^T                [dv, i]  Vc read MN-major
//   O2^T = S^T Qa^T                [dv, i]  S^T is a BF16 operand in tensor memory
//   T^T  = V'^T Kb                 [dv, dk] V' = lam^. Vc as three BF16 terms in tensor memory, Kb MN-major
//   out  = O1 + scale lam^. O2,    S <- lam^n S + T
// The state itself stays in registers in FP32.  Roundings to BF16: P and the copy of S that is read (one
// rounding each, as large as the output's own); V' is split into three terms (24 bits), so that T, and with
// it the state over any number of chunks, is exact to FP32.
//
// Roles (16 warps): 0-7 carry the state (thread = value column, half of the key columns) and scale V',
// 8-11 the outputs, 12-13 P, 14 TMA, 15 MMA.  V' is made and T issued in two halves of 32 tokens, so that the
// scaling of one overlaps the product of the other; O2, O1 and the next A run while the state warps take T.
// V' is in tensor memory because shared memory's bandwidth is what the products and copies share: as a
// shared-memory operand it took 768 more of its cycles per chunk (and 4100 cycles per chunk instead of 2900).
// Every wait is bounded; one that gives up sets the status bit and lets the CTA drain.
#include "decay_walk.cuh"
#include "tcgen05.cuh"

#include <cuda.h>

#include <mutex>

namespace bdm {
namespace {

using namespace walk;

constexpr int kThreads = 512;
constexpr int kBox = 64 * 128;  // bytes of a TMA box: 64 tokens x 64 BF16 columns
constexpr int kStateWarps = 8, kOutWarp = 8, kScoreWarp = 12, kTmaWarp = 14, kMmaWarp = 15;
constexpr int kMaxStages = 8;
constexpr int kSmemMax = 227 * 1024;
constexpr long long kWaitCycles = 4000000000ll;  // about 2 s
constexpr unsigned long long kWaitNs = 2000000000ull;

// tensor memory columns
constexpr uint32_t kColA = 0, kColO1 = 64, kColO2 = 128, kColT = 192, kColS = 320, kColV = 384;

struct Maps {
    CUtensorMap a, b, c, out;
};
struct TcParams {
    Params p;
    int amul[3], bmul[3];  // 0 where the operand's batch (head) is shared by all: a, b, c
};

struct Bars {
    uint64_t full[kMaxStages], empty[kMaxStages];
    uint64_t vready[2], tpart[2], sready, adone, pready, odone, ofree, zeroed, ofull, oempty;
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
// Two values as three BF16 terms each.
__device__ __forceinline__ void three_terms(F2 x, uint32_t &hi, uint32_t &mid, uint32_t &lo) {
    const F2 minus = make2(-1.f, -1.f);
    hi = pack2(x);
    x = fma2(unpack2(hi), minus, x);
    mid = pack2(x);
    x = fma2(unpack2(mid), minus, x);
    lo = pack2(x);
}

__device__ __noinline__ bool wait_slow(uint64_t *m, unsigned parity, volatile int *dead) {
    const long long t0 = clock64();
    for (int i = 0; i < (1 << 28); ++i) {
        if (tc::mbar_test_for(m, parity, 1000)) return true;
        if ((i & 15) == 15 && (*dead || clock64() - t0 > kWaitCycles)) break;
    }
    *dead = 1;
    return false;
}

// The state the segment starts from, key columns [k0, k0 + KC) of value column `col` (see start_state).
template <int KC>
__device__ __forceinline__ void start_states(const Params &p, const Span &s, int64_t bh, int seg, float g, int k0, int col,
                                             float (&S)[KC]) {
    const int64_t size = (int64_t)p.wab * p.wc;
    if (p.nseg > 1) {
        const float step = expf(g * (float)((int64_t)p.cps * kChunk));
        const int far = p.reverse ? (int)((s.chunks + p.cps - 1) / p.cps) - 1 : 0;
        const int count = p.reverse ? far - seg : seg;
        const float *z = p.seg + (bh * p.nseg + far) * size + (int64_t)col * p.wab + k0;
        for (int q = 0; q < count; ++q, z += p.reverse ? -size : size)
#pragma unroll
            for (int i = 0; i < KC; ++i)
                if (k0 + i < p.wab) S[i] = fmaf(S[i], step, z[i]);
    }
    if (p.state_in) {
        const int64_t end = s.c1 * kChunk < s.n ? s.c1 * kChunk : s.n;
        const int64_t far = p.reverse ? s.n - end : s.c0 * kChunk;
        const float w = (far ? expf(g * (float)far) : 1.f) * p.in_mul;
        const float *x = p.state_in + bh * size;
#pragma unroll
        for (int i = 0; i < KC; ++i)
            if (k0 + i < p.wab)
                S[i] = fmaf(w, x[p.in_t ? (int64_t)col * p.wab + k0 + i : (int64_t)(k0 + i) * p.wc + col], S[i]);
    }
}

// Stages of the load pipeline: what shared memory holds beside P and two buffers of outputs.
template <int DKB, int VB, bool STATE_ONLY> constexpr int stages_of() {
    const int stage = (STATE_ONLY ? DKB + VB : 2 * DKB + VB) * kBox;
    const int n = (kSmemMax - 1024 - 3072 - (1 + 2 * VB) * kBox) / stage;
    return n > kMaxStages ? kMaxStages : n;
}

// DKB, VB: 64-column boxes of a / b and of c.
template <int DKB, int VB, typename OT, bool STATE_ONLY>
__global__ void __launch_bounds__(kThreads, 1) decay_walk_tc_kernel(const TcParams tp, const __grid_constant__ Maps maps) {
    extern __shared__ char raw[];
    __shared__ Bars bar;
    __shared__ float pw[kChunk + 1], spw[kChunk + 1];  // lam^m, scale lam^m
    __shared__ float ow[2 * kChunk];                   // scale lam^. of a full chunk's tokens reading the state
    __shared__ float vw[2 * kChunk];                   // lam^. of a full chunk's tokens writing it
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int dead;
    const Params &p = tp.p;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    char *smem = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    constexpr int kStage = (STATE_ONLY ? DKB + VB : 2 * DKB + VB) * kBox;
    constexpr int kOffB = STATE_ONLY ? 0 : DKB * kBox, kOffC = kOffB + DKB * kBox;
    constexpr int DK = DKB * 64;
    constexpr int stages = stages_of<DKB, VB, STATE_ONLY>();
    char *sP = smem + stages * kStage;

    int64_t id = blockIdx.x;
    const int seg = (int)(id % p.nseg);
    const int64_t bh = id / p.nseg;
    const int64_t b = bh / p.heads;
    const int h = (int)(bh % p.heads);
    const float g = head_log_decay(p, h);
    const Span sp = span_of(p, row_tokens(p, b), seg);
    const int steps = (int)(sp.c1 - sp.c0);

    if (threadIdx.x <= kChunk) {
        pw[threadIdx.x] = threadIdx.x ? expf(g * (float)threadIdx.x) : 1.f;
        spw[threadIdx.x] = p.scale * pw[threadIdx.x];
    }
    if (threadIdx.x < 2 * kChunk) {  // a chunk with fewer tokens starts later in the tables that count down
        const int e = p.reverse ? kChunk - 1 - (int)threadIdx.x : (int)threadIdx.x + 1;
        ow[threadIdx.x] = e < 0 || e > kChunk ? 0.f : p.scale * (e ? expf(g * (float)e) : 1.f);
        const int f = p.reverse ? (int)threadIdx.x + 1 : kChunk - 1 - (int)threadIdx.x;
        vw[threadIdx.x] = f < 0 || f > kChunk ? 0.f : (f ? expf(g * (float)f) : 1.f);
    }
    if (threadIdx.x == 0) {
        dead = 0;
        for (int i = 0; i < stages; ++i) {
            tc::mbar_init(&bar.full[i], 1);
            tc::mbar_init(&bar.empty[i], 1);
        }
        tc::mbar_init(&bar.vready[0], kStateWarps);
        tc::mbar_init(&bar.vready[1], kStateWarps);
        tc::mbar_init(&bar.tpart[0], 1);
        tc::mbar_init(&bar.sready, kStateWarps);
        tc::mbar_init(&bar.tpart[1], 1);
        tc::mbar_init(&bar.adone, 1);
        tc::mbar_init(&bar.pready, 2);
        tc::mbar_init(&bar.odone, 1);
        tc::mbar_init(&bar.ofree, 4);
        tc::mbar_init(&bar.zeroed, kStateWarps);
        tc::mbar_init(&bar.ofull, 4);
        tc::mbar_init(&bar.oempty, 1);
        tc::mbar_fence_init();
    }
    if (warp == kMmaWarp) tc::tmem_alloc(&tmem_slot, 512);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = tmem_slot;

    // bounded waits, the second for a whole warp with one answer for its lanes; false once any has given up
    auto wait = [&](uint64_t *m, unsigned parity) -> bool { return tc::mbar_test(m, parity) || wait_slow(m, parity, &dead); };
    auto wait_warp = [&](uint64_t *m, unsigned parity) -> bool { return __all_sync(0xffffffffu, wait(m, parity)); };
    // first token and valid tokens of the n-th chunk of the walk
    const int tokens = (int)sp.n, time = (int)p.time;
    const int first = (int)(p.reverse ? sp.c1 - 1 : sp.c0) * kChunk, stride = p.reverse ? -kChunk : kChunk;
    auto start_of = [&](int n) -> int { return first + n * stride; };
    auto valid_of = [&](int n) -> int { return min(tokens - start_of(n), kChunk); };

    if (warp < kStateWarps) {
        // ------------------------------------------------------- V' and the state
        const int quad = warp & 3, half = warp >> 2;
        const int col = quad * 32 + lane;                  // value column = tensor-memory lane
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        constexpr int KC = DK / 2;                         // key columns of this thread
        const int k0 = half * KC;
        const bool mine = quad < 2 * VB;
        F2 S[KC / 2];
        {
            float x[KC];
#pragma unroll
            for (int i = 0; i < KC; ++i) x[i] = 0.f;
            if (!STATE_ONLY && col < p.wc) start_states<KC>(p, sp, bh, seg, g, k0, col, x);
#pragma unroll
            for (int i = 0; i < KC / 2; ++i) S[i] = make2(x[2 * i], x[2 * i + 1]);
        }
        bool ok = true;
        int valid = 0, before = 0;  // valid tokens of the chunk and of the one before
        int st = 0, phase = 0;  // stage of the chunk, parity of its barrier
        // this lane's row of the matrices it loads: two of 8 tokens by two of 8 columns
        const int mrow = ((lane >> 4) * 8 + (lane & 7)) * 128, mcol = (lane >> 3) & 1;
        auto arrive = [&](uint64_t *m) {
            tc::tmem_wait_st();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(m);
        };
        // Half steps (32 tokens) of a chunk; one copy of the scaling code, for the instruction cache's sake.
        for (int hs = 0; hs <= 2 * steps; ++hs) {
            const int n = hs >> 1, hb = hs & 1;
            if (hb == 0 && n < steps) {
                valid = valid_of(n);
                ok = wait_warp(&bar.full[st], phase);
                if (!ok) break;
                if (valid < kChunk && start_of(n) + valid < time) {
                    // tokens past the row's length may hold anything: zero them for the products over j
                    uint4 *kb = reinterpret_cast<uint4 *>(smem + st * kStage + kOffB);
#pragma unroll 1
                    for (int i = threadIdx.x; i < (DKB + VB) * kBox / 16; i += kStateWarps * 32)
                        if ((i % (kBox / 16)) / 8 >= valid) kb[i] = make_uint4(0, 0, 0, 0);
                    tc::fence_async_smem();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&bar.zeroed);  // once at most: a row has one such chunk
                    ok = wait_warp(&bar.zeroed, 0);
                    if (!ok) break;
                }
                if (n > 0) {
                    ok = wait_warp(&bar.tpart[0], (n - 1) & 1);
                    if (!ok) break;
                    tc::fence_after_sync();
                }
            }
            if (mine && n < steps) {
                // 16 tokens of V' from 32 hb + 16 half on, this quadrant's columns: transposed on the way in, scaled,
                // and split into BF16 terms as the fragments that tensor memory takes
                const int j0 = hb * 32 + half * 16;
                const char *src = smem + st * kStage + kOffC + (quad >> 1) * kBox + j0 * 128 + mrow;
                const float *w = vw + (p.reverse ? 0 : kChunk - valid) + j0 + 2 * (lane & 3);
                const F2 w0 = make2(w[0], w[1]), w1 = make2(w[8], w[9]);
#pragma unroll 1
                for (int d = 0; d < 2; ++d) {
                    uint32_t r[4], t[3][4];
                    tc::ldmatrix_x4_trans(src + ((((quad & 1) * 4 + d * 2 + mcol) ^ (lane & 7)) << 4), r);
#pragma unroll
                    for (int m = 0; m < 4; ++m) three_terms(mul2(m < 2 ? w0 : w1, unpack2(r[m])), t[0][m], t[1][m], t[2][m]);
#pragma unroll
                    for (int u = 0; u < 3; ++u)
                        tc::tmem_st_16x128b_x2(tmem + lanes + (d << 20) + kColV + hb * 48 + u * 16 + half * 8, t[u][0], t[u][1],
                                               t[u][2], t[u][3]);
                }
            }
            if (hb == 0) {
                if (n > 0) {
                    ok = wait_warp(&bar.tpart[1], (n - 1) & 1);
                    if (!ok) break;
                    tc::fence_after_sync();
                    if (mine) {
                        const F2 carry = make2(pw[before], pw[before]);
#pragma unroll
                        for (int i = 0; i < KC; i += 16) {
                            float t[16];
                            tc::tmem_ld16(tmem + lanes + kColT + k0 + i, t);
                            tc::tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 8; ++e) S[i / 2 + e] = fma2(carry, S[i / 2 + e], make2(t[2 * e], t[2 * e + 1]));
                        }
                    }
                }
                before = valid;
                if (n == steps) break;
                arrive(&bar.vready[0]);
            } else {
                arrive(&bar.vready[1]);
                if (++st == stages) st = 0, phase ^= 1;
                if (!STATE_ONLY) {
                    if (n > 0) {
                        ok = wait_warp(&bar.odone, (n - 1) & 1);  // the last chunk's reads of S are over
                        if (!ok) break;
                        tc::fence_after_sync();
                    }
                    if (mine)
#pragma unroll
                        for (int i = 0; i < KC; i += 32) {
                            uint32_t r[16];
#pragma unroll
                            for (int e = 0; e < 16; ++e) r[e] = pack2(S[i / 2 + e]);
                            tc::tmem_st16(tmem + lanes + kColS + (k0 + i) / 2, r);
                        }
                    arrive(&bar.sready);
                }
            }
        }
        if (ok && col < p.wc) {
            const int64_t size = (int64_t)p.wab * p.wc;
            auto at = [&](int i) { return i & 1 ? split2(S[i / 2]).y : split2(S[i / 2]).x; };
            if (STATE_ONLY) {
                float *z = p.seg + (bh * p.nseg + seg) * size + (int64_t)col * p.wab;
#pragma unroll
                for (int i = 0; i < KC; ++i)
                    if (k0 + i < p.wab) z[k0 + i] = at(i);
            } else if (p.state_out && sp.last) {
                float *z = p.state_out + bh * size;
#pragma unroll
                for (int i = 0; i < KC; ++i)
                    if (k0 + i < p.wab)
                        z[p.out_t ? (int64_t)col * p.wab + k0 + i : (int64_t)(k0 + i) * p.wc + col] = at(i) * p.out_mul;
            }
        }
    } else if (warp < kScoreWarp) {
        // ------------------------------------------------------------- outputs
        if constexpr (!STATE_ONLY) {
            const int quad = warp & 3;
            const int col = quad * 32 + lane;
            const uint32_t lanes = (uint32_t)(quad * 32) << 16;
            const bool on = col < p.wc;
            OT *out = static_cast<OT *>(p.out) + b * p.os[0] + h * p.os[2];
            constexpr bool kTma = sizeof(OT) == 2;  // BF16 outputs leave by TMA, FP32 ones (partial sums) by plain stores
            const int mtok = ((lane >> 4) * 8 + (lane & 7)) * 128, mcol = (lane >> 3) & 1;
            for (int n = 0; n < steps; ++n) {
                const int t0 = start_of(n), valid = valid_of(n);
                char *stage = sP + (1 + (n & 1) * VB) * kBox;  // BF16 outputs on their way, [token][column]: the map's boxes
                if (kTma && n > 1) {
                    if (warp == kOutWarp && lane == 0) {
                        tc::tma_store_wait_read<1>();
                        tc::mbar_arrive(&bar.oempty);
                    }
                    if (!wait_warp(&bar.oempty, n & 1)) break;
                }
                if (!wait_warp(&bar.odone, n & 1)) break;
                tc::fence_after_sync();
                if (quad < 2 * VB) {
                    const float *w0 = ow + (p.reverse ? kChunk - valid : 0) + 2 * (lane & 3);
                    // 16 columns by 32 tokens at a time.  Fragments: this lane has tokens 8 b + 2 (lane % 4) + {0, 1} of
                    // column 16 d + lane / 4 (+ 8).
#pragma unroll 1
                    for (int q = 0; q < 4; ++q) {
                        const int d = q >> 1, i = q & 1;
                        float y[16], z[16];
                        const uint32_t at = tmem + lanes + (d << 20) + i * 32;
                        tc::tmem_ld_16x256b_x4(at + kColO2, y);
                        tc::tmem_ld_16x256b_x4(at + kColO1, z);
                        const float *w = w0 + i * 32;
                        F2 wt[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) wt[e] = make2(w[8 * e], w[8 * e + 1]);
                        tc::tmem_wait_ld();
                        F2 x[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            x[e] = fma2(wt[e / 2], make2(y[2 * e], y[2 * e + 1]), make2(z[2 * e], z[2 * e + 1]));
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
                            char *dst = stage + (quad >> 1) * kBox + i * 32 * 128 + mtok +
                                        ((((quad & 1) * 4 + d * 2 + mcol) ^ (lane & 7)) << 4);
                            tc::stmatrix_x4_trans(dst, v[0], v[1], v[2], v[3]);
                            tc::stmatrix_x4_trans(dst + 16 * 128, v[4], v[5], v[6], v[7]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const int r = r0 + e / 2 * 8, c = quad * 32 + d * 16 + (e & 1) * 8 + (lane >> 2);
                                const float2 v = split2(x[e]);
                                OT *o = out + (int64_t)(t0 + r) * p.os[1] + c;
                                if (c < p.wc && t0 + r < time) o[0] = r < valid ? v.x : 0.f;
                                if (c < p.wc && t0 + r + 1 < time) o[p.os[1]] = r + 1 < valid ? v.y : 0.f;
                            }
                        }
                    }
                }
                tc::fence_before_sync();
                if (kTma) tc::fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    tc::mbar_arrive(&bar.ofree);
                    if (kTma) tc::mbar_arrive(&bar.ofull);
                }
                if (kTma && warp == kOutWarp) {
                    if (!wait_warp(&bar.ofull, n & 1)) break;
                    if (lane == 0) {
#pragma unroll
                        for (int i = 0; i < VB; ++i) tc::tma_store_4d(&maps.out, stage + i * kBox, i * 64, t0, h, (int)b);
                        tc::tma_store_commit();
                    }
                }
            }
            if (kTma && warp == kOutWarp && lane == 0) tc::tma_store_wait();
            // whole chunks past the row's length
            int64_t z0 = sp.chunks * kChunk, z1 = p.time;
            const int64_t s0 = (int64_t)seg * p.cps * kChunk, s1 = s0 + (int64_t)p.cps * kChunk;
            if (z0 < s0) z0 = s0;
            if (z1 > s1) z1 = s1;
            if (on)
                for (int64_t t = z0; t < z1; ++t) out[t * p.os[1] + col] = Elem<OT>::from_float(0.f);
        }
    } else if (warp < kTmaWarp) {
        // -------------------------------------------------- decayed scores P (rows 0..63)
        if constexpr (!STATE_ONLY) {
            const int quad = warp & 3;  // 0 or 1
            const int row = quad * 32 + lane;
            const uint32_t lanes = (uint32_t)(quad * 32) << 16;
            F2 w[32];  // the row's weights
#pragma unroll
            for (int j = 0; j < 64; j += 2) {
                const int d0 = p.reverse ? j - row : row - j, d1 = p.reverse ? d0 + 1 : d0 - 1;
                w[j / 2] = make2(d0 >= 0 ? spw[d0 < 0 ? 0 : d0] : 0.f, d1 >= 0 ? spw[d1 < 0 ? 0 : d1] : 0.f);
            }
            for (int n = 0; n < steps; ++n) {
                const int valid = valid_of(n);
                if (!wait_warp(&bar.adone, n & 1)) break;
                tc::fence_after_sync();
                uint32_t r[32];
#pragma unroll
                for (int i = 0; i < 64; i += 16) {
                    float x[16];
                    tc::tmem_ld16(tmem + lanes + kColA + i, x);
                    tc::tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; e += 2) r[(i + e) / 2] = pack2(mul2(w[(i + e) / 2], make2(x[e], x[e + 1])));
                }
                if (valid < kChunk)  // scores of tokens past the row's length may be anything
#pragma unroll
                    for (int j = 0; j < 64; j += 2)
                        r[j / 2] &= (j < valid ? 0xffffu : 0u) | (j + 1 < valid ? 0xffff0000u : 0u);
                if (n > 0 && !wait_warp(&bar.odone, (n - 1) & 1)) break;
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    *reinterpret_cast<uint4 *>(sP + row * 128 + ((c ^ (row & 7)) << 4)) =
                        make_uint4(r[4 * c], r[4 * c + 1], r[4 * c + 2], r[4 * c + 3]);
                tc::fence_async_smem();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&bar.pready);
            }
        }
    } else if (warp == kTmaWarp) {
        // ------------------------------------------------------------------ loads
        if (tc::elect_one()) {
            int issued = 0;
            int st = 0, phase = 0;
            for (int n = 0; n < steps; ++n) {
                if (n >= stages && !wait(&bar.empty[st], phase ^ 1)) break;
                char *dst = smem + st * kStage;
                const int t0 = start_of(n);
                tc::mbar_arrive_expect_tx(&bar.full[st], kStage);
                if (!STATE_ONLY)
#pragma unroll
                    for (int i = 0; i < DKB; ++i)
                        tc::tma_load_4d(dst + i * kBox, &maps.a, i * 64, t0, (h / p.ag) * tp.bmul[0], (int)b * tp.amul[0],
                                        &bar.full[st]);
#pragma unroll
                for (int i = 0; i < DKB; ++i)
                    tc::tma_load_4d(dst + kOffB + i * kBox, &maps.b, i * 64, t0, (h / p.bg) * tp.bmul[1],
                                    (int)b * tp.amul[1], &bar.full[st]);
#pragma unroll
                for (int i = 0; i < VB; ++i)
                    tc::tma_load_4d(dst + kOffC + i * kBox, &maps.c, i * 64, t0, (h / p.cg) * tp.bmul[2],
                                    (int)b * tp.amul[2], &bar.full[st]);
                issued = n + 1;
                if (++st == stages) st = 0, phase ^= 1;
            }
            // no copy may be in flight when the CTA ends, whatever happened to its consumers
            for (int n = issued > stages ? issued - stages : 0; n < issued; ++n)
                tc::mbar_wait(&bar.full[n % stages], (n / stages) & 1, kWaitNs);
        }
    } else {
        // --------------------------------------------------------------- products
        if (tc::elect_one()) {
            constexpr uint32_t idQK = tc::idesc_bf16(128, 64);
            constexpr uint32_t idO1 = tc::idesc_bf16(128, 64) | tc::kIdescMnA;
            constexpr uint32_t idO2 = tc::idesc_bf16(128, 64);
            constexpr uint32_t idT = tc::idesc_bf16(128, DK) | tc::kIdescMnB;
            // descriptors of the buffers' starts; an offset adds its bytes / 16 to the low word
            const uint32_t base = tc::smem_u32(smem);
            const uint64_t dP = tc::smem_desc_sw128(tc::smem_u32(sP));
            // rows 64..127 of the scores, and value columns past c's boxes, are whatever follows the tile
            auto scores = [&](int st) {
                uint64_t qa = tc::smem_desc_sw128(base + st * kStage), kb = qa + kOffB / 16;
#pragma unroll 1
                for (int i = 0; i < DKB; ++i, qa += kBox / 16, kb += kBox / 16)
#pragma unroll
                    for (int k = 0; k < 4; ++k) tc::mma_bf16(tmem + kColA, qa + k * 2, kb + k * 2, idQK, i + k > 0);
                tc::mma_commit(&bar.adone);
            };
            bool ok = true;
            int done = 0, st = 0, phase = 0;
            if (!STATE_ONLY && steps > 0) {
                ok = wait(&bar.full[0], 0);
                if (ok) scores(0);
            }
            for (int n = 0; n < steps && ok; ++n) {
                const uint32_t tile = base + st * kStage;
                uint64_t kb = tc::smem_desc_sw128_mn(tile + kOffB, kBox);
                uint32_t va = tmem + kColV;
#pragma unroll 1
                for (int hb = 0; hb < 2; ++hb, kb += 2 * 2048 / 16, va += 48) {
                    if (!(ok = wait(&bar.vready[hb], n & 1))) break;
                    tc::fence_after_sync();
#pragma unroll
                    for (int t = 0; t < 3; ++t)
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            tc::mma_bf16_tmem_a(tmem + kColT, va + t * 16 + k * 8, kb + k * 2048 / 16, idT, hb + t + k > 0);
                    tc::mma_commit(&bar.tpart[hb]);
                }
                if (!ok) break;
                if (!STATE_ONLY) {
                    if (!(ok = wait(&bar.sready, n & 1))) break;
                    if (n > 0 && !(ok = wait(&bar.ofree, (n - 1) & 1))) break;
                    tc::fence_after_sync();
                    uint64_t qa = tc::smem_desc_sw128(tile);
                    uint32_t sa = tmem + kColS;
#pragma unroll 1
                    for (int i = 0; i < DKB; ++i, qa += kBox / 16, sa += 32)
#pragma unroll
                        for (int k = 0; k < 4; ++k) tc::mma_bf16_tmem_a(tmem + kColO2, sa + k * 8, qa + k * 2, idO2, i + k > 0);
                    if (!(ok = wait(&bar.pready, n & 1))) break;
                    tc::fence_after_sync();
                    const uint64_t vc = tc::smem_desc_sw128_mn(tile + kOffC, kBox);
#pragma unroll
                    for (int k = 0; k < 4; ++k) tc::mma_bf16(tmem + kColO1, vc + k * 2048 / 16, dP + k * 2, idO1, k > 0);
                    tc::mma_commit(&bar.odone);
                }
                tc::mma_commit(&bar.empty[st]);
                done = n + 1;
                if (++st == stages) st = 0, phase ^= 1;
                if (!STATE_ONLY && n + 1 < steps) {
                    if (!(ok = wait(&bar.full[st], phase))) break;
                    scores(st);
                }
            }
            // nor a product
            if (done) tc::mbar_wait(&bar.empty[(done - 1) % stages], ((done - 1) / stages) & 1, kWaitNs);
        }
    }
    __syncwarp();
    tc::fence_before_sync();
    __syncthreads();
    if (threadIdx.x == 0 && dead && p.status) *(volatile int *)p.status = 0x4;
    if (warp == kMmaWarp) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, 512);
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static EncodeTiled fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return static_cast<EncodeTiled>(nullptr);
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return fn;
}

struct Operand {
    const void *ptr;
    const int64_t *stride;
    int width, heads;
};

// Columns, tokens, heads, batch; a dimension every index of which is the same memory becomes one of size 1.
bool fits_tma(const Operand &o, int64_t time, int64_t batch) {
    if (reinterpret_cast<uintptr_t>(o.ptr) & 15) return false;
    const int64_t size[3] = {batch, time, o.heads};
    for (int i = 0; i < 3; ++i) {
        if (size[i] == 1) continue;
        if (o.stride[i] == 0 && i != 1) continue;
        if (o.stride[i] <= 0 || o.stride[i] % 8 || o.stride[i] * 2 >= ((int64_t)1 << 40)) return false;
        if (size[i] > 0x7fffffff) return false;
    }
    return true;
}
bool encode(EncodeTiled fn, CUtensorMap *m, const Operand &o, int64_t time, int64_t batch, int &amul, int &bmul) {
    amul = batch > 1 && o.stride[0] != 0;
    bmul = o.heads > 1 && o.stride[2] != 0;
    const cuuint64_t dims[4] = {(cuuint64_t)o.width, (cuuint64_t)time, (cuuint64_t)(bmul ? o.heads : 1),
                                (cuuint64_t)(amul ? batch : 1)};
    const cuuint64_t any = ((cuuint64_t)o.width * 2 + 15) / 16 * 16;  // of dimensions of size 1: nothing uses it
    const cuuint64_t strides[3] = {time > 1 ? (cuuint64_t)o.stride[1] * 2 : any, bmul ? (cuuint64_t)o.stride[2] * 2 : any,
                                   amul ? (cuuint64_t)o.stride[0] * 2 : any};
    const cuuint32_t box[4] = {64, kChunk, 1, 1}, estr[4] = {1, 1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(o.ptr), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DKB, int VB, typename OT, bool STATE_ONLY> int launch(TcParams &tp, const Maps &maps, cudaStream_t st) {
    const int smem = stages_of<DKB, VB, STATE_ONLY>() * (STATE_ONLY ? DKB + VB : 2 * DKB + VB) * kBox + (1 + 2 * VB) * kBox + 1024;
    auto kernel = decay_walk_tc_kernel<DKB, VB, OT, STATE_ONLY>;
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
            set[dev] = true;
        }
    }
    const int64_t blocks = tp.p.batch * tp.p.heads * tp.p.nseg;
    if (blocks > 0x7fffffff) return BDM_ERR_UNSUPPORTED;
    kernel<<<(unsigned)blocks, kThreads, smem, st>>>(tp, maps);
    return launch_status();
}

template <int DKB, int VB> int launch_types(TcParams &tp, const Maps &maps, bool out_f32, bool state_only, cudaStream_t st) {
    if (state_only) return launch<DKB, VB, bf16, true>(tp, maps, st);
    if (out_f32) return launch<DKB, VB, float, false>(tp, maps, st);
    return launch<DKB, VB, bf16, false>(tp, maps, st);
}

}  // namespace

bool decay_walk_tc_takes(const bdm_decay_walk_args &w) {
    if (w.dtype != BDM_BF16 || w.time <= 0 || w.time > 0x7fffffff - kChunk) return false;
    const Operand ops[3] = {{w.a, w.a_stride, w.width_ab, w.a_heads},
                            {w.b, w.b_stride, w.width_ab, w.b_heads},
                            {w.c, w.c_stride, w.width_c, w.c_heads}};
    for (const Operand &o : ops)
        if (!fits_tma(o, w.time, w.batch)) return false;
    if (w.out_dtype == BDM_BF16) {
        if (!fits_tma({w.out, w.out_stride, w.width_c, w.heads}, w.time, w.batch)) return false;
        if ((w.batch > 1 && !w.out_stride[0]) || (w.heads > 1 && !w.out_stride[2])) return false;
    }
    return encode_tiled() != nullptr;
}

// Segments of the time axis: the count that makes the two launches shortest, in units of one chunk of the
// main walk.  A CTA has an SM to itself; its start and end cost about three chunks, a chunk of the state
// launch about half of one, and a segment start reads all its predecessors' states.
int64_t decay_walk_tc_segments(int64_t rows, int64_t chunks, int sms) {
    int64_t best = 1;
    double cost = 0;
    for (int64_t s = 1; s <= chunks / 4 + 1 && s <= 64 && (s == 1 || rows * (s - 1) < sms); ++s) {
        const int64_t cps = ceil_div(chunks, s), waves = ceil_div(rows * s, sms);
        const double c = waves * (cps + 3.0 + (s > 1 ? 0.5 * cps + 5.0 + 0.2 * s : 0.0));
        if (s == 1 || c < cost) cost = c, best = s;
    }
    return best;
}

int decay_walk_tc_launch(const bdm_decay_walk_args &w, const Params &p, bool state_only, cudaStream_t st) {
    EncodeTiled fn = encode_tiled();
    if (!fn) return BDM_ERR_UNSUPPORTED;
    TcParams tp{};
    tp.p = p;
    Maps maps;
    const Operand ops[3] = {{w.a, w.a_stride, w.width_ab, w.a_heads},
                            {w.b, w.b_stride, w.width_ab, w.b_heads},
                            {w.c, w.c_stride, w.width_c, w.c_heads}};
    CUtensorMap *m[3] = {&maps.a, &maps.b, &maps.c};
    for (int i = 0; i < 3; ++i)
        if (!encode(fn, m[i], ops[i], w.time, w.batch, tp.amul[i], tp.bmul[i])) return BDM_ERR_UNSUPPORTED;
    if (w.out_dtype == BDM_BF16) {
        int amul, bmul;
        if (!encode(fn, &maps.out, {w.out, w.out_stride, w.width_c, w.heads}, w.time, w.batch, amul, bmul))
            return BDM_ERR_UNSUPPORTED;
    }
    const bool f32 = w.out_dtype == BDM_F32;
    if (p.wab > 64) {
        if (p.wc > 64) return launch_types<2, 2>(tp, maps, f32, state_only, st);
        return launch_types<2, 1>(tp, maps, f32, state_only, st);
    }
    if (p.wc > 64) return launch_types<1, 2>(tp, maps, f32, state_only, st);
    return launch_types<1, 1>(tp, maps, f32, state_only, st);
}

}  // namespace bdm
