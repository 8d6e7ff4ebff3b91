// Decay attention, one token per row: S <- lam S + k v^T (in place, FP32), o = scale q S.
//
// The state is read and written once (8 dk dv bytes per head) and nothing else matters: the bound is HBM (256
// rows of 8 heads of 128: 44 us, 41 at the copy rate).
// A CTA owns one (row, head) and a slice of dv columns; a thread holds 4 columns (one 16-byte access) of
// every 8th..32nd state row, all its loads are issued before the first use, and the partial sums of o over
// the state's rows are joined in shared memory in a fixed order.
#include "decay_walk.cuh"

namespace bdm {
namespace {

constexpr int kThreads = 256;
constexpr int kBatchRows = 4;  // state rows a thread loads at a time

// VEC columns per thread (4 where dv and the state allow 16-byte accesses, else 1); LANES threads cover a
// slice of LANES * VEC columns, kThreads / LANES state rows are processed side by side.
template <typename T, int VEC, int LANES>
__global__ void __launch_bounds__(kThreads)
    decay_step_kernel(const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, int64_t qsb, int64_t qsh,
                      int64_t ksb, int64_t ksh, int64_t vsb, int64_t vsh, int group, const float *__restrict__ log_decay,
                      float *__restrict__ state, T *__restrict__ out, int heads, int dk, int dv, float scale, int slices) {
    constexpr int kRows = kThreads / LANES;
    __shared__ float red[kRows][LANES * VEC];
    extern __shared__ float qk[];  // q [dk], k [dk]
    const int slice = (int)(blockIdx.x % slices);
    const int64_t bh = blockIdx.x / slices;
    const int64_t b = bh / heads;
    const int h = (int)(bh % heads);
    const int lane = threadIdx.x % LANES, row = threadIdx.x / LANES;
    const int col = (slice * LANES + lane) * VEC;
    const bool in = col < dv;
    float *s = state + bh * dk * dv + col;
    const float g = log_decay[h];
    const float lam = expf(g);
    // the first state rows are on their way while q, k and v are read
    float S[kBatchRows][VEC];
    auto fetch = [&](int i0) {
#pragma unroll
        for (int u = 0; u < kBatchRows; ++u) {
            const int i = i0 + u * kRows;
            if (in && i < dk) {
                if constexpr (VEC == 4) {
                    const float4 x = *reinterpret_cast<const float4 *>(s + (int64_t)i * dv);
                    S[u][0] = x.x, S[u][1] = x.y, S[u][2] = x.z, S[u][3] = x.w;
                } else {
                    S[u][0] = s[(int64_t)i * dv];
                }
            }
        }
    };
    fetch(row);
    for (int i = threadIdx.x; i < dk; i += kThreads) {
        qk[i] = Elem<T>::to_float(q[b * qsb + h * qsh + i]);
        qk[dk + i] = Elem<T>::to_float(k[b * ksb + (h / group) * ksh + i]);
    }
    float vv[VEC], o[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        vv[e] = col + e < dv ? Elem<T>::to_float(v[b * vsb + (h / group) * vsh + col + e]) : 0.f;
        o[e] = 0.f;
    }
    __syncthreads();
    for (int i0 = row; i0 < dk; i0 += kBatchRows * kRows) {
        if (i0 != row) fetch(i0);
#pragma unroll
        for (int u = 0; u < kBatchRows; ++u) {
            const int i = i0 + u * kRows;
            if (!in || i >= dk) continue;
            const float qi = qk[i], ki = qk[dk + i];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                S[u][e] = fmaf(lam, S[u][e], ki * vv[e]);
                o[e] = fmaf(qi, S[u][e], o[e]);
            }
            if constexpr (VEC == 4)
                *reinterpret_cast<float4 *>(s + (int64_t)i * dv) = make_float4(S[u][0], S[u][1], S[u][2], S[u][3]);
            else
                s[(int64_t)i * dv] = S[u][0];
        }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) red[row][lane * VEC + e] = o[e];
    __syncthreads();
    for (int j = threadIdx.x; j < LANES * VEC; j += kThreads) {
        const int c = slice * LANES * VEC + j;
        if (c >= dv) continue;
        float x = 0.f;
#pragma unroll 8
        for (int r = 0; r < kRows; ++r) x += red[r][j];
        out[bh * dv + c] = Elem<T>::from_float(x * scale);
    }
}

template <typename T>
int launch(const bdm_decay_step_args &a, cudaStream_t st) {
    const bool vec = a.value_width % 4 == 0 && (reinterpret_cast<uintptr_t>(a.state) & 15) == 0;
    const int64_t bh = a.batch * a.heads;
    const int smem = 2 * a.key_width * (int)sizeof(float);
#define BDM_STEP(VEC, LANES)                                                                                          \
    do {                                                                                                              \
        const int slices = (int)ceil_div(a.value_width, VEC * LANES);                                                 \
        if (bh * slices > 0x7fffffff) return BDM_ERR_UNSUPPORTED;                                                     \
        decay_step_kernel<T, VEC, LANES><<<(unsigned)(bh * slices), kThreads, smem, st>>>(                            \
            static_cast<const T *>(a.q), static_cast<const T *>(a.k), static_cast<const T *>(a.v), a.q_stride[0],     \
            a.q_stride[1], a.k_stride[0], a.k_stride[1], a.v_stride[0], a.v_stride[1], a.heads / a.kv_heads,          \
            a.log_decay, a.state, static_cast<T *>(a.out), a.heads, a.key_width, a.value_width, a.scale, slices);     \
    } while (0)
    if (!vec)
        BDM_STEP(1, 32);
    else if (a.value_width > 64)
        BDM_STEP(4, 32);
    else if (a.value_width > 32)
        BDM_STEP(4, 16);
    else
        BDM_STEP(4, 8);
#undef BDM_STEP
    return launch_status();
}

}  // namespace
}  // namespace bdm

extern "C" int bdm_decay_step(const bdm_decay_step_args *a, void *stream) {
    using namespace bdm;
    if (!a || a->batch < 0 || a->heads <= 0 || a->kv_heads <= 0 || a->heads % a->kv_heads || a->key_width <= 0 ||
        a->value_width <= 0)
        return BDM_ERR_INVALID;
    if (!valid_dtype(a->dtype)) return BDM_ERR_DTYPE;
    if (a->key_width > 1024) return BDM_ERR_UNSUPPORTED;
    if (a->batch == 0) return BDM_OK;
    if (!a->q || !a->k || !a->v || !a->log_decay || !a->state || !a->out) return BDM_ERR_INVALID;
    if (a->dtype == BDM_F32) return launch<float>(*a, as_stream(stream));
    return launch<bf16>(*a, as_stream(stream));
}
