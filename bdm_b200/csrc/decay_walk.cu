// Decay attention (linear attention with a decay for each head): the walk over a row's tokens on FP32
// CUDA cores, the sum of shared heads' gradients, and the C entry points.
//
// The walk's mathematics is in decay_walk.cuh.  This kernel takes every type and stride: operands are
// widened to FP32 in shared memory and all products, sums and states are FP32.
#include "decay_walk.cuh"

#include <mutex>

namespace bdm {
namespace {

using namespace walk;

constexpr int kThreads = 256;
constexpr int kCols = 64;  // columns of c per CTA

// Shared memory (floats): A, B [64][wab+4], Cc [64][64], P [64][68], S [wab][64], powers [65].
int simt_smem(int wab, bool state_only) {
    const int pitch = ((wab + 3) & ~3) + 4;
    int f = kChunk * pitch + kChunk * kCols + kChunk + 4;
    if (!state_only) f += kChunk * pitch + kChunk * (kChunk + 4) + ((wab + 3) & ~3) * kCols;
    return f * 4;
}

// Rows [t0, t0 + 64) of one head into shared memory as FP32; invalid rows and columns are zero.  A warp takes
// every 8th row, its lanes neighbouring columns; four rows' loads are in flight at a time.
template <typename T>
__device__ __forceinline__ void load_rows(float *dst, int pitch, const T *src, int64_t st, int64_t t0, int valid, int first,
                                          int width, int cols) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int d = lane; d < cols; d += 32) {
        const bool in = first + d < width;
        const T *p = src + t0 * st + first + d;
#pragma unroll
        for (int u0 = 0; u0 < kChunk / 8; u0 += 4) {
            float x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int r = warp + (u0 + u) * 8;
                x[u] = in && r < valid ? Elem<T>::to_float(p[r * st]) : 0.f;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) dst[(warp + (u0 + u) * 8) * pitch + d] = x[u];
        }
    }
}

// One CTA walks one segment of one (row, head) for 64 columns of c.
template <typename T, typename OT, bool STATE_ONLY>
__global__ void __launch_bounds__(kThreads) decay_walk_kernel(const Params p) {
    extern __shared__ float sm[];
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
    const int wk = (p.wab + 3) & ~3, pitch = wk + 4;
    const int n0 = slice * kCols;

    float *sB = sm;
    float *sC = sB + kChunk * pitch;
    float *pw = sC + kChunk * kCols;  // lam^0 .. lam^64
    float *sA = pw + kChunk + 4;
    float *sP = sA + kChunk * pitch;
    float *sS = sP + kChunk * (kChunk + 4);

    const float g = head_log_decay(p, h);
    for (int i = threadIdx.x; i <= kChunk; i += kThreads) pw[i] = i ? expf(g * (float)i) : 1.f;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    if (!STATE_ONLY && p.nseg > 1) asm volatile("griddepcontrol.wait;\n" ::: "memory");

    const Span sp = span_of(p, row_tokens(p, b), seg);
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const T *a = static_cast<const T *>(p.a) + b * p.as[0] + (h / p.ag) * p.as[2];
    const T *bb = static_cast<const T *>(p.b) + b * p.bs[0] + (h / p.bg) * p.bs[2];
    const T *c = static_cast<const T *>(p.c) + b * p.cs[0] + (h / p.cg) * p.cs[2];
    OT *out = static_cast<OT *>(p.out) + b * p.os[0] + h * p.os[2];

    // state elements (ty + 16 r, n0 + 4 tx + e) in registers
    const int64_t size = (int64_t)p.wab * p.wc;
    const bool before = !STATE_ONLY && p.nseg > 1 && (p.reverse ? seg < p.nseg - 1 : seg > 0);
    float given = 0.f;
    if (!STATE_ONLY && p.state_in) {
        const int64_t end = sp.c1 * kChunk < sp.n ? sp.c1 * kChunk : sp.n;
        const int64_t far = p.reverse ? sp.n - end : sp.c0 * kChunk;
        given = (far ? expf(g * (float)far) : 1.f) * p.in_mul;
    }
    float S[8][4];
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = ty + 16 * r, j = n0 + 4 * tx + e;
            S[r][e] = 0.f;
            if (i >= p.wab || j >= p.wc) continue;
            if (before) S[r][e] = p.seg[(bh * p.nseg + seg) * size + (int64_t)i * p.wc + j];
            if (!STATE_ONLY && p.state_in)
                S[r][e] = fmaf(given, p.state_in[bh * size + (p.in_t ? (int64_t)j * p.wab + i : (int64_t)i * p.wc + j)], S[r][e]);
        }

    for (int64_t step = 0; step < sp.c1 - sp.c0; ++step) {
        const int64_t ch = p.reverse ? sp.c1 - 1 - step : sp.c0 + step;
        const int64_t t0 = ch * kChunk;
        const int valid = (int)(sp.n - t0 < kChunk ? sp.n - t0 : kChunk);
        __syncthreads();  // the tiles of the previous chunk are done with
        if (!STATE_ONLY) {
            load_rows<T>(sA, pitch, a, p.as[1], t0, valid, 0, p.wab, wk);
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (ty + 16 * r < wk) *reinterpret_cast<float4 *>(&sS[(ty + 16 * r) * kCols + 4 * tx]) =
                    make_float4(S[r][0], S[r][1], S[r][2], S[r][3]);
        }
        load_rows<T>(sB, pitch, bb, p.bs[1], t0, valid, 0, p.wab, wk);
        load_rows<T>(sC, kCols, c, p.cs[1], t0, valid, n0, p.wc, kCols);
        __syncthreads();

        if (!STATE_ONLY) {
            // P = (A B^T) with the decay between the rows; rows ty + 16 r, columns tx + 16 q
            float acc[4][4] = {};
            for (int k = 0; k < wk; k += 4) {
                float4 x[4], y[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = *reinterpret_cast<const float4 *>(&sA[(ty + 16 * r) * pitch + k]);
#pragma unroll
                for (int q = 0; q < 4; ++q) y[q] = *reinterpret_cast<const float4 *>(&sB[(tx + 16 * q) * pitch + k]);
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        acc[r][q] += x[r].x * y[q].x + x[r].y * y[q].y + x[r].z * y[q].z + x[r].w * y[q].w;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int i = ty + 16 * r, j = tx + 16 * q;
                    const int d = p.reverse ? j - i : i - j;
                    sP[i * (kChunk + 4) + j] = d >= 0 ? acc[r][q] * pw[d] : 0.f;
                }
            __syncthreads();
            // out = scale * (P C + lam^. A S); rows ty + 16 r, columns 4 tx .. 4 tx + 3
            float o[4][4] = {};
            for (int k = 0; k < wk; k += 4) {
                float4 x[4], y[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = *reinterpret_cast<const float4 *>(&sA[(ty + 16 * r) * pitch + k]);
#pragma unroll
                for (int q = 0; q < 4; ++q) y[q] = *reinterpret_cast<const float4 *>(&sS[(k + q) * kCols + 4 * tx]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    o[r][0] += x[r].x * y[0].x + x[r].y * y[1].x + x[r].z * y[2].x + x[r].w * y[3].x;
                    o[r][1] += x[r].x * y[0].y + x[r].y * y[1].y + x[r].z * y[2].y + x[r].w * y[3].y;
                    o[r][2] += x[r].x * y[0].z + x[r].y * y[1].z + x[r].z * y[2].z + x[r].w * y[3].z;
                    o[r][3] += x[r].x * y[0].w + x[r].y * y[1].w + x[r].z * y[2].w + x[r].w * y[3].w;
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = ty + 16 * r;
                const int e = p.reverse ? valid - 1 - i : i + 1;
                const float w = e >= 0 ? pw[e] : 0.f;
#pragma unroll
                for (int q = 0; q < 4; ++q) o[r][q] *= w;
            }
            for (int j = 0; j < kChunk; j += 4) {
                float4 x[4], y[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = *reinterpret_cast<const float4 *>(&sP[(ty + 16 * r) * (kChunk + 4) + j]);
#pragma unroll
                for (int q = 0; q < 4; ++q) y[q] = *reinterpret_cast<const float4 *>(&sC[(j + q) * kCols + 4 * tx]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    o[r][0] += x[r].x * y[0].x + x[r].y * y[1].x + x[r].z * y[2].x + x[r].w * y[3].x;
                    o[r][1] += x[r].x * y[0].y + x[r].y * y[1].y + x[r].z * y[2].y + x[r].w * y[3].y;
                    o[r][2] += x[r].x * y[0].z + x[r].y * y[1].z + x[r].z * y[2].z + x[r].w * y[3].z;
                    o[r][3] += x[r].x * y[0].w + x[r].y * y[1].w + x[r].z * y[2].w + x[r].w * y[3].w;
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = ty + 16 * r;
                if (t0 + i >= p.time) continue;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int j = n0 + 4 * tx + q;
                    if (j < p.wc)
                        out[(t0 + i) * p.os[1] + j] = Elem<OT>::from_float(i < valid ? p.scale * o[r][q] : 0.f);
                }
            }
        }
        // S = lam^valid S + sum_j lam^. b_j c_j, where anyone asks for it
        if (!STATE_ONLY && step + 1 == sp.c1 - sp.c0 && !(p.state_out && sp.last)) break;
        const float carry = pw[valid];
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[r][e] *= carry;
        for (int j = 0; j < valid; ++j) {
            float4 y = *reinterpret_cast<const float4 *>(&sC[j * kCols + 4 * tx]);
            const float w = pw[p.reverse ? j + 1 : valid - 1 - j];
            y.x *= w, y.y *= w, y.z *= w, y.w *= w;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                if (ty + 16 * r >= wk) continue;
                const float x = sB[j * pitch + ty + 16 * r];
                S[r][0] += x * y.x, S[r][1] += x * y.y, S[r][2] += x * y.z, S[r][3] += x * y.w;
            }
        }
    }

    if (STATE_ONLY || (p.state_out && sp.last)) {
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = ty + 16 * r, j = n0 + 4 * tx + e;
                if (i >= p.wab || j >= p.wc) continue;
                if (STATE_ONLY)
                    p.seg[(bh * segs + zid) * size + (int64_t)i * p.wc + j] = S[r][e];
                else
                    p.state_out[bh * size + (p.out_t ? (int64_t)j * p.wab + i : (int64_t)i * p.wc + j)] =
                        S[r][e] * p.out_mul;
            }
    }
    if (!STATE_ONLY) {
        // rows of whole chunks past the row's length
        int64_t z0 = sp.chunks * kChunk, z1 = p.time;
        const int64_t s0 = (int64_t)seg * p.cps * kChunk, s1 = s0 + (int64_t)p.cps * kChunk;
        if (z0 < s0) z0 = s0;
        if (z1 > s1) z1 = s1;
        const int cols = p.wc - n0 < kCols ? p.wc - n0 : kCols;
        for (int64_t i = threadIdx.x; i < (z1 - z0) * cols; i += kThreads)
            out[(z0 + i / cols) * p.os[1] + n0 + i % cols] = Elem<OT>::from_float(0.f);
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
    std::lock_guard<std::mutex> lock(g_mu);
    if (!g_attr[dev]) {
        const void *fns[] = {
            (const void *)decay_walk_kernel<float, float, false>, (const void *)decay_walk_kernel<float, float, true>,
            (const void *)decay_walk_kernel<bf16, bf16, false>, (const void *)decay_walk_kernel<bf16, float, false>,
            (const void *)decay_walk_kernel<bf16, bf16, true>};
        for (const void *f : fns)
            if (int rc = cuda_status(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                          simt_smem(kMaxWidth, false))))
                return rc;
        if (int rc = cuda_status(cudaDeviceGetAttribute(&g_sms[dev], cudaDevAttrMultiProcessorCount, dev))) return rc;
        g_attr[dev] = true;
    }
    sms = g_sms[dev];
    return BDM_OK;
}

// The state launch, the prefix launch and the walk; each start overlaps the end of the one before.
template <typename T, typename OT> int simt_launch(Params p, void *workspace, cudaStream_t st) {
    const int64_t rows = p.batch * p.heads, slices = ceil_div(p.wc, kCols), size = (int64_t)p.wab * p.wc;
    if (rows * slices * p.nseg > 0x7fffffff) return BDM_ERR_UNSUPPORTED;
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(kThreads);
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
        cfg.dynamicSmemBytes = simt_smem(p.wab, true);
        if (int rc = cuda_status(cudaLaunchKernelEx(&cfg, decay_walk_kernel<T, T, true>, (const Params)q))) return rc;
        if (int rc = launch_status()) return rc;
        if (int rc = decay_prefix_launch(p, z, 1, p.cps, st)) return rc;
        cfg.numAttrs = 1;
    }
    cfg.gridDim = dim3((unsigned)(rows * slices * p.nseg));
    cfg.dynamicSmemBytes = simt_smem(p.wab, false);
    if (int rc = cuda_status(cudaLaunchKernelEx(&cfg, decay_walk_kernel<T, OT, false>, (const Params)p))) return rc;
    return launch_status();
}

// Segments of the time axis for the CUDA-core walk: three CTAs per SM, down to a chunk each.  A segment more
// costs a second pass over its b and c and half of a chunk's arithmetic, so rows that fill the GPU stay whole.
int64_t simt_segments(int64_t ctas, int64_t chunks, int sms) {
    if (ctas >= 2 * sms) return 1;
    const int64_t s = 3 * sms / ctas;
    return s > chunks ? chunks : s;
}

struct Split {
    bool tc;        // the tensor-core walk takes it
    int sub, scps;  // its state launch's sub-segments and their chunks
};

int plan(const bdm_decay_walk_args &w, Params &p, Split &split, int sms) {
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
    split = Split{decay_walk_tc_takes(w), 1, 1};
    if (split.tc) {
        decay_walk_tc_split(w.batch * w.heads, chunks, sms, p.nseg, p.cps, split.sub, split.scps);
    } else {
        const int64_t nseg = simt_segments(w.batch * w.heads * ceil_div(w.width_c, kCols), chunks, sms);
        p.cps = (int)ceil_div(chunks, nseg);
        p.nseg = (int)ceil_div(chunks, p.cps);
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

int64_t seg_bytes(const Params &p, const Split &split) {
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
    Split split{};
    if (plan(*w, p, split, sms)) return -1;
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
    Split split{};
    if (int rc = plan(*w, p, split, sms)) return rc;
    const int64_t need = seg_bytes(p, split);
    if (need > workspace_bytes || (need && !workspace)) return BDM_ERR_WORKSPACE;
    cudaStream_t st = as_stream(stream);
    if (split.tc) return decay_walk_tc_launch(*w, p, split.sub, split.scps, workspace, st);
    if (w->dtype == BDM_F32) return simt_launch<float, float>(p, workspace, st);
    if (w->out_dtype == BDM_F32) return simt_launch<bf16, float>(p, workspace, st);
    return simt_launch<bf16, bf16>(p, workspace, st);
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
