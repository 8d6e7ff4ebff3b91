// Decay attention (linear attention with a decay for each head): the walk over a row's tokens for FP32 operands
// and for BF16 ones that TMA cannot address, the sum of shared heads' gradients, and the C entry points.
//
// The walk's mathematics is in decay_walk.cuh.  Operands are widened to FP32 in shared memory.  Every product
// a b runs on the tensor cores as three TF32 products, a1 b1 + a1 b2 + a2 b1 with a = a1 + a2 + r, |r| <= 2^-22 |a|
// (the method of splitting an operand into its rounding and the remainder), summed in FP32: about 3e-7 beside
// FP32's own 1e-7, where plain TF32 gives 5e-4.  Sums and states are FP32.  Bound: the TF32 products' rate and
// the latency of a chunk's phases (2 x 4096 tokens x 8 heads of 128: 354 us; 3 x 777 x 6 heads of 40 / 72: 48 us
// in three launches, on FP32 FMAs with the same tiles 72).
#include "decay_walk.cuh"

#include <mutex>

namespace bdm {
namespace {

using namespace walk;

constexpr int kCols = 64;  // columns of c per CTA

constexpr int kColPitch = kCols + 8;    // C, S: 8 banks from row to row
constexpr int kScorePitch = kChunk + 4;  // P (as A, B): 4 banks
__host__ __device__ constexpr int walk_width(int wab) { return (wab + 15) & ~15; }

// Shared memory (floats): B [64][w+4], C [64][72], powers [68], A [64][w+4], P [64][68], S [w][72].
int walk_smem(int wab, bool state_only) {
    const int w = walk_width(wab), pitch = w + 4;
    int f = kChunk * pitch + kChunk * kColPitch + kChunk + 4;
    if (!state_only) f += kChunk * pitch + kChunk * kScorePitch + w * kColPitch;
    return f * 4;
}

// x = big + small, both TF32 operands (the tensor core drops the bits of `small` past TF32's).  An infinite x makes
// its products NaN: what it reaches is not finite either way.
struct Split32 {
    uint32_t big, small;
};
__device__ __forceinline__ Split32 split32(float x) {
    Split32 s;
    asm("cvt.rna.tf32.f32 %0, %1;\n" : "=r"(s.big) : "f"(x));
    s.small = __float_as_uint(x - __uint_as_float(s.big));
    return s;
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d[n] += a (16 x 8) b (8 x 8, columns 8 n), n < N.  a(i): element i of this lane's fragment (rows g, g + 8, then
// the same rows 4 columns on); b(n, i): element i of tile n (rows t, t + 4).  g = lane / 4, t = lane % 4.
template <int N, typename FA, typename FB> __device__ __forceinline__ void mma_step(float (&d)[N][4], FA a, FB b) {
    uint32_t big[4], small[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const Split32 s = split32(a(i));
        big[i] = s.big, small[i] = s.small;
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const Split32 b0 = split32(b(n, 0)), b1 = split32(b(n, 1));
        // The tensor core cuts its sums off rather than rounding them: over a long sum that is a drift (2.5e-6 after
        // 20000 tokens).  So its sums are of 8 products, and they are added up by FP32 additions.
        float t[4] = {};
        mma_tf32(t, small, b0.big, b1.big);
        mma_tf32(t, big, b0.small, b1.small);
        mma_tf32(t, big, b0.big, b1.big);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[n][i] += t[i];
    }
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// Rows [t0, t0 + 64) of one head into shared memory as FP32; invalid rows and columns are zero.  A warp takes
// every WARPS-th row, its lanes neighbouring columns; four rows' loads are in flight at a time.  Returns NaN
// where one of this thread's values is infinite or NaN, else 0.
template <int WARPS, typename T>
__device__ __forceinline__ float load_rows(float *dst, int pitch, const T *src, int64_t st, int64_t t0, int valid, int first,
                                          int width, int cols) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float odd = 0.f;
    for (int d = lane; d < cols; d += 32) {
        const bool in = first + d < width;
        const T *p = src + t0 * st + first + d;
#pragma unroll
        for (int u0 = 0; u0 < kChunk / WARPS; u0 += 4) {
            float x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int r = warp + (u0 + u) * WARPS;
                x[u] = in && r < valid ? Elem<T>::to_float(p[r * st]) : 0.f;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) odd = fmaf(x[u], 0.f, odd);
#pragma unroll
            for (int u = 0; u < 4; ++u) dst[(warp + (u0 + u) * WARPS) * pitch + d] = x[u];
        }
    }
    return odd;
}

// One CTA walks one segment of one (row, head) for 64 columns of c.  With 8 warps, P and the outputs are 4 x 2
// warp tiles of 16 x 32 and a warp has two of the state's up to 8 x 2 tiles of that size; with 16 warps, 4 x 4 of
// 16 x 16 and one of the state's.  Shared memory decides: up to 80 columns of a and b two or three CTAs of 8 warps
// share an SM (3 x 777 x 6 heads of 40 / 72: 48 us, with 16 warps 55), past that one of 16 hides more latency than
// one of 8 (2 x 4096 x 8 heads of 128: 354 us, with 8 warps 430, issuing in 38 % of the cycles).
template <int WARPS, typename T, typename OT, bool STATE_ONLY>
__global__ void __launch_bounds__(WARPS * 32) decay_walk_kernel(const Params p) {
    constexpr int kThreads = WARPS * 32, N = 32 / WARPS, ST = 16 / WARPS;
    extern __shared__ float sm[];
    __shared__ int odd_step;         // the last step that met a c that is not finite
    __shared__ int odd_from[kCols];  // of a chunk where c is not finite: each column's first such row (reverse: last)
    const int slices = (p.wc + kCols - 1) / kCols;
    int64_t id = blockIdx.x;
    const int segs = STATE_ONLY ? p.nseg - 1 : p.nseg;
    const int zid = (int)(id % segs);
    const int seg = STATE_ONLY ? zid + p.reverse : zid;  // the last segment walked needs no state of its own
    id /= segs;
    const int slice = (int)(id % slices);
    const int64_t bh = id / slices;
    const int64_t b = bh / p.heads;
    const int h = (int)(bh % p.heads);
    const int width = walk_width(p.wab), pitch = width + 4;
    const int n0 = slice * kCols;

    float *sB = sm;
    float *sC = sB + kChunk * pitch;
    float *pw = sC + kChunk * kColPitch;  // lam^0 .. lam^64
    float *sA = pw + kChunk + 4;
    float *sP = sA + kChunk * pitch;
    float *sS = sP + kChunk * kScorePitch;

    const float g = head_log_decay(p, h);
    for (int i = threadIdx.x; i <= kChunk; i += kThreads) pw[i] = i ? expf(g * (float)i) : 1.f;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    if (!STATE_ONLY && p.nseg > 1) asm volatile("griddepcontrol.wait;\n" ::: "memory");

    const Span sp = span_of(p, row_tokens(p, b), seg);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lg = lane >> 2, lt = lane & 3;
    const int mrow = (warp & 3) * 16, ncol = (warp >> 2) * 8 * N;  // this warp's tile of P and of the outputs
    const T *a = static_cast<const T *>(p.a) + b * p.as[0] + (h / p.ag) * p.as[2];
    const T *bb = static_cast<const T *>(p.b) + b * p.bs[0] + (h / p.bg) * p.bs[2];
    const T *c = static_cast<const T *>(p.c) + b * p.cs[0] + (h / p.cg) * p.cs[2];
    OT *out = static_cast<OT *>(p.out) + b * p.os[0] + h * p.os[2];
    const int64_t size = (int64_t)p.wab * p.wc;

    // state tile q: rows srow(q) + lg (+ 8), columns scol + 8 n + 2 lt + {0, 1}; element (n, i) is row lg + 8 (i / 2)
    const int scol = warp % 2 * 32;
    auto srow = [&](int q) { return (warp + WARPS * q) / 2 * 16; };
    float S[ST][4][4];
    {
        const bool before = !STATE_ONLY && p.nseg > 1 && (p.reverse ? seg < p.nseg - 1 : seg > 0);
        const float *zs = before ? p.seg + (bh * p.nseg + seg) * size : nullptr;
        const float *x = !STATE_ONLY && p.state_in ? p.state_in + bh * size : nullptr;
        float given = 0.f;
        if (x) {
            const int64_t end = sp.c1 * kChunk < sp.n ? sp.c1 * kChunk : sp.n;
            const int64_t far = p.reverse ? sp.n - end : sp.c0 * kChunk;
            given = (far ? expf(g * (float)far) : 1.f) * p.in_mul;
        }
#pragma unroll
        for (int q = 0; q < ST; ++q)
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int k = srow(q) + lg + 8 * (i >> 1), v = n0 + scol + 8 * n + 2 * lt + (i & 1);
                    const bool in = k < p.wab && v < p.wc;
                    S[q][n][i] = 0.f;
                    if (zs) {
                        const float f = zs[in ? k * p.wc + v : 0];
                        S[q][n][i] = in ? f : 0.f;
                    }
                    if (x) {
                        const float f = x[in ? (p.in_t ? v * p.wab + k : k * p.wc + v) : 0];
                        S[q][n][i] = in ? fmaf(given, f, S[q][n][i]) : 0.f;
                    }
                }
    }

    if (threadIdx.x == 0) odd_step = -1;
    for (int64_t step = 0; step < sp.c1 - sp.c0; ++step) {
        const int64_t ch = p.reverse ? sp.c1 - 1 - step : sp.c0 + step;
        const int64_t t0 = ch * kChunk;
        const int valid = (int)(sp.n - t0 < kChunk ? sp.n - t0 : kChunk);
        __syncthreads();  // the tiles of the previous chunk are done with
        if (!STATE_ONLY) {
            load_rows<WARPS, T>(sA, pitch, a, p.as[1], t0, valid, 0, p.wab, width);
#pragma unroll
            for (int q = 0; q < ST; ++q)
                if (srow(q) < width)
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int i = 0; i < 4; i += 2)
                            *reinterpret_cast<float2 *>(&sS[(srow(q) + lg + 4 * i) * kColPitch + scol + 8 * n + 2 * lt]) =
                                make_float2(S[q][n][i], S[q][n][i + 1]);
        }
        load_rows<WARPS, T>(sB, pitch, bb, p.bs[1], t0, valid, 0, p.wab, width);
        const float odd = load_rows<WARPS, T>(sC, kColPitch, c, p.cs[1], t0, valid, n0, p.wc, kCols);
        if (!STATE_ONLY && odd != odd) odd_step = (int)step;
        __syncthreads();
        const bool odd_chunk = !STATE_ONLY && odd_step == (int)step;
        if (odd_chunk) {
            // c has values that are not finite, which a masked score of zero would turn into NaN: they count as zero in
            // the product with the scores.  What they do reach, the column's outputs from there on, is set to NaN after
            // it, and so is the value that the state takes in.
            if (threadIdx.x < kCols) {
                float *col = sC + threadIdx.x;
                int from = p.reverse ? -1 : kChunk;
                for (int r = 0; r < kChunk; ++r)
                    if (!finite(col[r * kColPitch])) {
                        from = p.reverse ? r : min(from, r);
                        col[r * kColPitch] = 0.f;
                    }
                odd_from[threadIdx.x] = from;
            }
            __syncthreads();
        }

        if (!STATE_ONLY) {
            // P = A B^T with the decay between the rows; tiles that the mask empties are only cleared
            float d[N][4] = {};
            if (p.reverse ? ncol + 8 * N - 1 >= mrow : ncol <= mrow + 15) {
                const float *fa = sA + (mrow + lg) * pitch + lt, *fb = sB + (ncol + lg) * pitch + lt;
#pragma unroll 2
                for (int k = 0; k < width; k += 8)
                    mma_step(d, [&](int i) { return fa[(i & 1) * 8 * pitch + (i >> 1) * 4 + k]; },
                             [&](int n, int i) { return fb[n * 8 * pitch + i * 4 + k]; });
            }
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const int r = mrow + lg + 4 * i, j = ncol + 8 * n + 2 * lt;
                    const int e0 = p.reverse ? j - r : r - j, e1 = p.reverse ? e0 + 1 : e0 - 1;
                    *reinterpret_cast<float2 *>(&sP[r * kScorePitch + j]) =
                        make_float2(e0 >= 0 ? d[n][i] * pw[e0] : 0.f, e1 >= 0 ? d[n][i + 1] * pw[e1] : 0.f);
                }
            __syncthreads();
            // out = scale * (lam^. A S + P C)
            float o[N][4] = {};
            {
                const float *fa = sA + (mrow + lg) * pitch + lt, *fs = sS + lt * kColPitch + ncol + lg;
#pragma unroll 2
                for (int k = 0; k < width; k += 8)
                    mma_step(o, [&](int i) { return fa[(i & 1) * 8 * pitch + (i >> 1) * 4 + k]; },
                             [&](int n, int i) { return fs[(k + i * 4) * kColPitch + n * 8]; });
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = mrow + lg + 8 * (i >> 1);
                const int e = p.reverse ? valid - 1 - r : r + 1;
                const float w = e >= 0 ? pw[e] : 0.f;
#pragma unroll
                for (int n = 0; n < N; ++n) o[n][i] *= w;
            }
            {
                const float *fp = sP + (mrow + lg) * kScorePitch + lt, *fc = sC + lt * kColPitch + ncol + lg;
                const int k0 = p.reverse ? mrow : 0, k1 = p.reverse ? kChunk : mrow + 16;  // outside, P is zero
#pragma unroll 2
                for (int k = k0; k < k1; k += 8)
                    mma_step(o, [&](int i) { return fp[(i & 1) * 8 * kScorePitch + (i >> 1) * 4 + k]; },
                             [&](int n, int i) { return fc[(k + i * 4) * kColPitch + n * 8]; });
            }
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = mrow + lg + 8 * (i >> 1), j = n0 + ncol + 8 * n + 2 * lt + (i & 1);
                    if (t0 + r < p.time && j < p.wc)
                        out[(t0 + r) * p.os[1] + j] = Elem<OT>::from_float(r < valid ? p.scale * o[n][i] : 0.f);
                }
            if (odd_chunk) {
                __syncthreads();
                const int col = threadIdx.x, from = col < kCols ? odd_from[col] : -1;
                if (from >= 0 && from < valid) {
                    sC[from * kColPitch + col] = NAN;
                    for (int r = p.reverse ? 0 : from; r < (p.reverse ? from + 1 : valid); ++r)
                        out[(t0 + r) * p.os[1] + n0 + col] = Elem<OT>::from_float(NAN);
                }
                __syncthreads();
            }
        }
        // S = lam^valid S + sum_j lam^. b_j c_j, where anyone asks for it
        if (!STATE_ONLY && step + 1 == sp.c1 - sp.c0 && !(p.state_out && sp.last)) break;
        const float carry = pw[valid];
#pragma unroll
        for (int q = 0; q < ST; ++q) {
            if (srow(q) >= width) continue;
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) S[q][n][i] *= carry;
            const float *fb = sB + lt * pitch + srow(q) + lg, *fc = sC + lt * kColPitch + scol + lg;
            for (int k = 0; k < valid; k += 8) {  // rows past `valid` are zero
                float w[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int e = p.reverse ? k + lt + 4 * i + 1 : valid - 1 - (k + lt + 4 * i);
                    w[i] = pw[e < 0 ? 0 : e];
                }
                mma_step(S[q], [&](int i) { return fb[(k + (i >> 1) * 4) * pitch + (i & 1) * 8]; },
                         [&](int n, int i) { return w[i] * fc[(k + i * 4) * kColPitch + n * 8]; });
            }
        }
    }

    if (STATE_ONLY || (p.state_out && sp.last)) {
        float *z = STATE_ONLY ? p.seg + (bh * segs + zid) * size : p.state_out + bh * size;
#pragma unroll
        for (int q = 0; q < ST; ++q)
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int k = srow(q) + lg + 8 * (i >> 1), v = n0 + scol + 8 * n + 2 * lt + (i & 1);
                    if (k >= p.wab || v >= p.wc) continue;
                    if (STATE_ONLY)
                        z[k * p.wc + v] = S[q][n][i];
                    else
                        z[p.out_t ? v * p.wab + k : k * p.wc + v] = S[q][n][i] * p.out_mul;
                }
    }
    if (!STATE_ONLY) {
        // rows of whole chunks past the row's length
        int64_t z0 = sp.chunks * kChunk, z1 = p.time;
        const int64_t s0 = (int64_t)seg * p.cps * kChunk, s1 = s0 + (int64_t)p.cps * kChunk;
        if (z0 < s0) z0 = s0;
        if (z1 > s1) z1 = s1;
        const int cols = p.wc - n0 < kCols ? p.wc - n0 : kCols;
        for (int64_t t = z0 + warp; t < z1; t += kThreads / 32)
            for (int j = lane; j < cols; j += 32) out[t * p.os[1] + n0 + j] = Elem<OT>::from_float(0.f);
    }
}

// The state each segment starts from (without the given one): the sub-segments before it in walk order, each
// lam^(tokens of one) further away than the next.  One thread per state element.
__global__ void __launch_bounds__(256) decay_prefix_kernel(const Params p, const float *__restrict__ z, int sub, int scps) {
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    const int64_t size = (int64_t)p.wab * p.wc, blocks = (size + 255) / 256;
    const int64_t bh = blockIdx.x / blocks, e = blockIdx.x % blocks * 256 + threadIdx.x;
    if (e >= size) return;
    const float step = expf(head_log_decay(p, (int)(bh % p.heads)) * (float)((int64_t)scps * kChunk));
    const int count = (p.nseg - 1) * sub;
    const int64_t dir = p.reverse ? -1 : 1;
    const float *src = z + (bh * count + (p.reverse ? count - 1 : 0)) * size + e;
    float *dst = p.seg + (bh * p.nseg + (p.reverse ? p.nseg - 2 : 1)) * size + e;
    float acc = 0.f;
    int u = 0;
    for (int i = 0; i < count; i += 8) {
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = i + k < count ? src[dir * (i + k) * size] : 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (i + k >= count) break;
            acc = fmaf(acc, step, x[k]);
            if (++u == sub) {
                *dst = acc;
                dst += dir * size;
                u = 0;
            }
        }
    }
}

// out[t, g, d] = sum over the group's heads of part[t, g * group + s, d] (FP32), in head order.
template <typename T>
__global__ void group_sum_kernel(const float *__restrict__ part, int64_t tokens, int groups, int group, int width,
                                 T *__restrict__ out) {
    const int64_t total = tokens * groups * width;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t tg = i / width;
        const int d = (int)(i % width);
        const float *src = part + tg * group * width + d;
        float x = 0.f;
        for (int s = 0; s < group; ++s) x += src[(int64_t)s * width];
        out[i] = Elem<T>::from_float(x);
    }
}

constexpr int kMaxDevices = 64;
std::mutex g_mu;
bool g_attr[kMaxDevices];
int g_sms[kMaxDevices];

int device_setup(int &sms) {
    int dev = 0;
    if (int rc = cuda_status(cudaGetDevice(&dev))) return rc;
    if (dev < 0 || dev >= kMaxDevices) return BDM_ERR_UNSUPPORTED;
    // a thread's first call (an autograd worker's) may come before anything has made the context current, which
    // encoding a tensor map needs
    if (int rc = cuda_status(cudaSetDevice(dev))) return rc;
    std::lock_guard<std::mutex> lock(g_mu);
    if (!g_attr[dev]) {
        const void *fns[] = {
            (const void *)decay_walk_kernel<8, float, float, false>, (const void *)decay_walk_kernel<16, float, float, false>,
            (const void *)decay_walk_kernel<8, bf16, bf16, false>,   (const void *)decay_walk_kernel<16, bf16, bf16, false>,
            (const void *)decay_walk_kernel<8, bf16, float, false>,  (const void *)decay_walk_kernel<16, bf16, float, false>,
            (const void *)decay_walk_kernel<8, float, float, true>,  (const void *)decay_walk_kernel<8, bf16, bf16, true>};
        for (const void *f : fns)
            if (int rc = cuda_status(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                          walk_smem(kMaxWidth, false))))
                return rc;
        if (int rc = cuda_status(cudaDeviceGetAttribute(&g_sms[dev], cudaDevAttrMultiProcessorCount, dev))) return rc;
        g_attr[dev] = true;
    }
    sms = g_sms[dev];
    return BDM_OK;
}

// The state launch, the prefix launch and the walk; each start overlaps the end of the one before.
template <typename T, typename OT> int walk_launch(Params p, void *workspace, cudaStream_t st) {
    const int64_t rows = p.batch * p.heads, slices = ceil_div(p.wc, kCols), size = (int64_t)p.wab * p.wc;
    if (rows * slices * p.nseg > 0x7fffffff) return BDM_ERR_UNSUPPORTED;
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    if (p.nseg > 1) {
        p.seg = static_cast<float *>(workspace);
        float *z = p.seg + rows * p.nseg * size;
        Params q = p;
        q.seg = z;
        cfg.gridDim = dim3((unsigned)(rows * slices * (p.nseg - 1)));
        cfg.dynamicSmemBytes = walk_smem(p.wab, true);
        if (int rc = cuda_status(cudaLaunchKernelEx(&cfg, decay_walk_kernel<8, T, T, true>, (const Params)q))) return rc;
        if (int rc = launch_status()) return rc;
        if (int rc = decay_prefix_launch(p, z, 1, p.cps, st)) return rc;
        cfg.numAttrs = 1;
    }
    cfg.gridDim = dim3((unsigned)(rows * slices * p.nseg));
    cfg.dynamicSmemBytes = walk_smem(p.wab, false);
    const bool wide = p.wab > 80;  // shared memory holds one CTA
    cfg.blockDim = dim3(wide ? 512 : 256);
    auto kernel = wide ? decay_walk_kernel<16, T, OT, false> : decay_walk_kernel<8, T, OT, false>;
    if (int rc = cuda_status(cudaLaunchKernelEx(&cfg, kernel, (const Params)p))) return rc;
    return launch_status();
}

// Segments of the time axis for this walk: three CTAs per SM, down to a chunk each.  A segment more
// costs a second pass over its b and c and half of a chunk's arithmetic, so rows that fill the GPU stay whole.
int64_t walk_segments(int64_t ctas, int64_t chunks, int sms) {
    if (ctas >= 2 * sms) return 1;
    const int64_t s = 3 * sms / ctas;
    return s > chunks ? chunks : s;
}

int plan(const bdm_decay_walk_args &w, Params &p, WalkSplit &split, bool &tc, int sms) {
    p.a = w.a, p.b = w.b, p.c = w.c, p.out = w.out;
    for (int i = 0; i < 3; ++i) {
        p.as[i] = w.a_stride[i];
        p.bs[i] = w.b_stride[i];
        p.cs[i] = w.c_stride[i];
        p.os[i] = w.out_stride[i];
    }
    p.ag = w.heads / w.a_heads, p.bg = w.heads / w.b_heads, p.cg = w.heads / w.c_heads;
    p.log_decay = w.log_decay;
    p.lengths = w.lengths;
    p.state_in = w.state_in, p.state_out = w.state_out;
    p.in_mul = w.state_in_mul, p.out_mul = w.state_out_mul;
    p.in_t = w.state_in_transposed, p.out_t = w.state_out_transposed;
    p.batch = w.batch, p.time = w.time;
    p.heads = w.heads, p.wab = w.width_ab, p.wc = w.width_c, p.reverse = w.reverse;
    p.scale = w.scale;
    p.status = w.status;
    p.seg = nullptr;
    const int64_t chunks = ceil_div(w.time, kChunk) > 0 ? ceil_div(w.time, kChunk) : 1;
    tc = decay_walk_tc_takes(w);
    if (tc) {
        split = decay_walk_tc_split(w.batch * w.heads, chunks, w.width_c, sms);
        p.nseg = split.nseg;
        p.cps = split.cps;
    } else {
        const int64_t nseg = walk_segments(w.batch * w.heads * ceil_div(w.width_c, kCols), chunks, sms);
        p.cps = (int)ceil_div(chunks, nseg);
        p.nseg = (int)ceil_div(chunks, p.cps);
        split = WalkSplit{p.nseg, p.cps, 1, p.cps, 1};
    }
    return BDM_OK;
}

int check_args(const bdm_decay_walk_args &w) {
    if (w.batch < 0 || w.time < 0 || w.heads <= 0 || w.width_ab <= 0 || w.width_c <= 0) return BDM_ERR_INVALID;
    if (w.a_heads <= 0 || w.b_heads <= 0 || w.c_heads <= 0) return BDM_ERR_INVALID;
    if (w.heads % w.a_heads || w.heads % w.b_heads || w.heads % w.c_heads) return BDM_ERR_INVALID;
    if (w.reverse != 0 && w.reverse != 1) return BDM_ERR_INVALID;
    if (!valid_dtype(w.dtype) || !valid_dtype(w.out_dtype)) return BDM_ERR_DTYPE;
    if (w.dtype == BDM_F32 && w.out_dtype != BDM_F32) return BDM_ERR_DTYPE;
    if (w.width_ab > kMaxWidth || w.width_c > kMaxWidth) return BDM_ERR_UNSUPPORTED;
    if (w.time > (int64_t)1 << 31) return BDM_ERR_UNSUPPORTED;
    return BDM_OK;
}

int64_t seg_bytes(const Params &p, const WalkSplit &split) {
    return p.nseg > 1 ? p.batch * p.heads * ((int64_t)p.nseg + (int64_t)(p.nseg - 1) * split.sub) * p.wab * p.wc * 4 : 0;
}

}  // namespace

int decay_prefix_launch(const walk::Params &p, const float *z, int sub, int scps, cudaStream_t st) {
    const int64_t blocks = p.batch * p.heads * ceil_div((int64_t)p.wab * p.wc, 256);
    if (blocks > 0x7fffffff) return BDM_ERR_UNSUPPORTED;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (int rc = cuda_status(cudaLaunchKernelEx(&cfg, decay_prefix_kernel, p, z, sub, scps))) return rc;
    return launch_status();
}

}  // namespace bdm

extern "C" int64_t bdm_decay_walk_workspace_bytes(const bdm_decay_walk_args *w) {
    using namespace bdm;
    if (!w || check_args(*w)) return -1;
    if (w->batch == 0) return 0;
    int sms = 0;
    if (device_setup(sms)) return -1;
    Params p{};
    WalkSplit split{};
    bool tc = false;
    if (plan(*w, p, split, tc, sms)) return -1;
    return seg_bytes(p, split);
}

extern "C" int bdm_decay_walk(const bdm_decay_walk_args *w, void *workspace, int64_t workspace_bytes, void *stream) {
    using namespace bdm;
    if (!w) return BDM_ERR_INVALID;
    if (int rc = check_args(*w)) return rc;
    if (w->batch == 0) return BDM_OK;
    if (!w->log_decay || (w->time > 0 && (!w->a || !w->b || !w->c || !w->out))) return BDM_ERR_INVALID;
    int sms = 0;
    if (int rc = device_setup(sms)) return rc;
    Params p{};
    WalkSplit split{};
    bool tc = false;
    if (int rc = plan(*w, p, split, tc, sms)) return rc;
    const int64_t need = seg_bytes(p, split);
    if (need > workspace_bytes || (need && !workspace)) return BDM_ERR_WORKSPACE;
    cudaStream_t st = as_stream(stream);
    if (tc) return decay_walk_tc_launch(*w, p, split, workspace, st);
    if (w->dtype == BDM_F32) return walk_launch<float, float>(p, workspace, st);
    if (w->out_dtype == BDM_F32) return walk_launch<bf16, float>(p, workspace, st);
    return walk_launch<bf16, bf16>(p, workspace, st);
}

extern "C" int bdm_decay_group_sum(const float *part, int64_t tokens, int groups, int group, int width, int dtype, void *out,
                                   void *stream) {
    using namespace bdm;
    if (tokens < 0 || groups <= 0 || group <= 0 || width <= 0) return BDM_ERR_INVALID;
    if (!valid_dtype(dtype)) return BDM_ERR_DTYPE;
    if (tokens == 0) return BDM_OK;
    if (!part || !out) return BDM_ERR_INVALID;
    int64_t blocks = ceil_div(tokens * groups * width, 256);
    if (blocks > 32 * kNumSMs) blocks = 32 * kNumSMs;
    BDM_DISPATCH_DTYPE(dtype, T, {
        group_sum_kernel<T><<<(unsigned)blocks, 256, 0, as_stream(stream)>>>(part, tokens, groups, group, width,
                                                                            static_cast<T *>(out));
    });
    return launch_status();
}
