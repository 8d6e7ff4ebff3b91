// Beam search: selection over beams x vocabulary, and the in-place reordering of decoder states.
#include "common.cuh"

namespace bdm {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxBeams = 32;
constexpr int64_t kMaxVocab = 0x7fff0000;  // token indices, rounded up to a whole slice, are ints
constexpr int kList = 1024;  // candidates a CTA collects before it falls back to repeated maxima

using u64 = unsigned long long;

// Order of floats as unsigned integers, -0 as +0; NaN never gets here.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
// Larger value first, then lower index; 0 is no candidate (its index would be 2^32 - 1 and its value NaN).
__device__ __forceinline__ u64 make_key(float x, uint32_t index) { return (u64)ordered(x) << 32 | (uint32_t)~index; }
__device__ __forceinline__ float key_value(u64 k) { return unordered((uint32_t)(k >> 32)); }
__device__ __forceinline__ uint32_t key_index(u64 k) { return ~(uint32_t)k; }

// Sorts one key per lane, largest in lane 0.
__device__ __forceinline__ u64 warp_sort_desc(u64 x) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int d = size >> 1; d > 0; d >>= 1) {
            const u64 y = __shfl_xor_sync(0xffffffffu, x, d);
            const bool up = (lane & size) == 0, low = (lane & d) == 0;
            x = (up == low) == (x > y) ? x : y;
        }
    return x;
}
__device__ __forceinline__ u64 warp_max(u64 x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 y = __shfl_xor_sync(0xffffffffu, x, o);
        x = x > y ? x : y;
    }
    return x;
}

struct TopShared {
    u64 list[kList];
    u64 best[kMaxBeams];
    u64 warp[kWarps];
    int count;
};

__device__ u64 block_max(u64 m, TopShared &sh) {
    m = warp_max(m);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = sh.warp[w] > m ? sh.warp[w] : m;
    return m;
}

// The K largest keys by K rounds of a CTA-wide maximum, in sh.best; each(use) calls use(key) for the thread's.
template <typename F> __device__ __forceinline__ void block_maxima(int K, TopShared &sh, F each) {
    u64 last = ~0ull;
    for (int r = 0; r < K; ++r) {
        u64 m = 0;
        each([&](u64 x) {
            if (x < last && x > m) m = x;
        });
        last = block_max(m, sh);
        if (threadIdx.x == 0) sh.best[r] = last;
        if (last == 0) break;
    }
    __syncthreads();
}

// ------------------------------------------------------------- per row slices

// Per (row, split): the slice's maximum, the sum of exp(x - max), and its K largest logits by (value,
// lower index).
struct Slice {
    float max, sum;
};

template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int n = 4;
};
template <> struct Vec<bf16> {
    static constexpr int n = 8;
};

template <typename T> __device__ __forceinline__ void unpack(const uint4 &r, float *x);
template <> __device__ __forceinline__ void unpack<float>(const uint4 &r, float *x) {
    x[0] = __uint_as_float(r.x), x[1] = __uint_as_float(r.y), x[2] = __uint_as_float(r.z), x[3] = __uint_as_float(r.w);
}
template <> __device__ __forceinline__ void unpack<bf16>(const uint4 &r, float *x) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

__device__ __forceinline__ float exp2_ftz(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

// Two FP32 values in one register pair, for the packed FP32 instructions.
__device__ __forceinline__ u64 pair(float x, float y) {
    u64 r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 halves(u64 a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
    u64 r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
    u64 r;
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// The slice's maximum and a lower bound of its K-th largest logit.  Every warp draws its K largest lane maxima
// (equal ones leave together: the bound is lower then, which is no harm).  For K <= 8 the bound is the K-th
// largest of all warps' together, which hardly more than K logits reach; past that, the largest of the warps'
// K-th largest, which several times K do.
__device__ __forceinline__ void slice_bound(float mine, int K, float *redm, float *redk, float &m, float &bound,
                                            TopShared &sh) {
    constexpr unsigned all = 0xffffffffu;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t *drawn = reinterpret_cast<uint32_t *>(sh.list);  // [warp][8], before the list is used
    uint32_t left = mine == mine ? ordered(mine) : 0u, kth = 0, top = 0;
    for (int k = 0; k < K; ++k) {
        kth = __reduce_max_sync(all, left);
        if (k == 0) top = kth;
        if (K <= 8 && lane == 0) drawn[warp * 8 + k] = kth;
        if (left == kth) left = 0;
    }
    if (lane == 0) {
        redm[warp] = unordered(top ? top : ordered(-INFINITY));
        redk[warp] = unordered(kth ? kth : ordered(-INFINITY));
    }
    if (threadIdx.x == 0) sh.count = 0;
    if (threadIdx.x < K) sh.best[threadIdx.x] = 0;
    __syncthreads();
    m = redm[0], bound = redk[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) {
        m = fmaxf(m, redm[w]);
        bound = fmaxf(bound, redk[w]);
    }
    if (K <= 8) {  // 64 values, two a lane
        uint32_t a = (lane & 7) < K ? drawn[lane] : 0u, b = (lane & 7) < K ? drawn[lane + 32] : 0u;
        for (int k = 0; k < K; ++k) {
            kth = __reduce_max_sync(all, a > b ? a : b);
            if (a == kth) a = 0;
            if (b == kth) b = 0;
        }
        bound = kth ? unordered(kth) : -INFINITY;
        __syncthreads();  // the list's memory is free
    }
}

// Joins the warps' sums, collects the candidates that hot(use) names by index (a logit is read again: registers
// have no index) and writes the K largest.
template <typename T, typename F>
__device__ __forceinline__ void finish_slice(float warp_total, float m, F hot, TopShared &sh, const T *src,
                                             int base, int count, int vocab, int K, Slice *stat, u64 *dst) {
    __shared__ float reds[kWarps];
    if ((threadIdx.x & 31) == 0) reds[threadIdx.x >> 5] = warp_total;
    hot([&](int i) {
        if (i >= vocab) return;
        const int at = atomicAdd(&sh.count, 1);
        if (at < kList) sh.list[at] = make_key(Elem<T>::to_float(src[i]), (uint32_t)i);
    });
    __syncthreads();
    if (threadIdx.x == 0) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) t += reds[w];
        *stat = Slice{t == t ? m : NAN, t};
    }
    const int n = sh.count;
    if (n <= kList) {
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const u64 k = sh.list[i];
            int rank = 0;
            for (int j = 0; j < n && rank < K; ++j) rank += sh.list[j] > k;
            if (rank < K) dst[rank] = k;
        }
        for (int i = n + threadIdx.x; i < K; i += kThreads) dst[i] = 0;
        return;
    }
    // a few threads hold most of the largest logits: repeated maxima, over the logits read again
    const int end = base + count < vocab ? base + count : vocab;
    block_maxima(K, sh, [&](auto &&use) {
#pragma unroll 1
        for (int i = base + threadIdx.x; i < end; i += kThreads) {
            const float y = Elem<T>::to_float(src[i]);
            if (y == y) use(make_key(y, (uint32_t)i));
        }
    });
    if (threadIdx.x < K) dst[threadIdx.x] = sh.best[threadIdx.x];
}

// One pass over the logits, E per thread in registers: the maximum, then the sum of exp(x - max) (one
// multiplication and ex2.approx: off by 2^-22, and by |x - max| 2^-24 for terms that are exp(x - max) small),
// then the few candidates: the logits at or above slice_bound's bound go to a list and are ranked there; when
// the list overflows, K rounds of a CTA-wide maximum take its place.  HBM is the floor (5 us for 64 x 8 x 32000
// BF16), instructions the bound: about 10 per logit and 300 per warp, 14 us.
// VECTOR: rows start on 16-byte boundaries.
template <typename T, int E, bool VECTOR>
__global__ void __launch_bounds__(kThreads)
    beam_slice_kernel(const T *__restrict__ logits, int64_t ld, int vocab, int K, int splits, Slice *__restrict__ stat,
                      u64 *__restrict__ lists) {
    __shared__ TopShared sh;
    __shared__ float redm[kWarps], redk[kWarps];
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const int64_t row = blockIdx.x / splits;
    const int split = (int)(blockIdx.x % splits);
    const int base = split * (E * kThreads);
    const T *src = logits + row * ld;
    constexpr int V = VECTOR ? Vec<T>::n : 1;
    float x[E];
    auto index = [&](int e) { return base + (e / V * kThreads + (int)threadIdx.x) * V + e % V; };
    if (VECTOR && base + E * kThreads <= vocab) {
        uint4 r[E / V];
#pragma unroll
        for (int e = 0; e < E / V; ++e) r[e] = *reinterpret_cast<const uint4 *>(src + index(e * V));
#pragma unroll
        for (int e = 0; e < E / V; ++e) unpack<T>(r[e], x + e * V);
    } else {
#pragma unroll
        for (int e = 0; e < E; e += V) {
            const int i = index(e);
            if (VECTOR && i + V <= vocab) {
                unpack<T>(*reinterpret_cast<const uint4 *>(src + i), x + e);
            } else {
#pragma unroll
                for (int u = 0; u < V; ++u) x[e + u] = i + u < vocab ? Elem<T>::to_float(src[i + u]) : -INFINITY;
            }
        }
    }
    float mine = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) mine = fmaxf(mine, x[e]);
    float m, bound;
    slice_bound(mine, K, redm, redk, m, bound, sh);
    // NaN and +inf make the sum NaN, and with it the whole row's log-probabilities
    float s0 = 0.f, s1 = 0.f;
    if (m > -INFINITY) {
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            s0 += exp2_ftz((x[e] - m) * 1.4426950408889634f);
            s1 += exp2_ftz((x[e + 1] - m) * 1.4426950408889634f);
        }
    } else {  // all -inf, or NaN
#pragma unroll
        for (int e = 0; e < E; ++e) s0 += x[e] == -INFINITY ? 0.f : NAN;
    }
    finish_slice<T>(warp_sum(s0 + s1), m, [&](auto &&use) {
        if (mine < bound) return;
        uint32_t hot = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) hot |= x[e] >= bound ? 1u << e : 0u;
        for (; hot; hot &= hot - 1) use(index(__ffs(hot) - 1));
    }, sh, src, base, E * kThreads, vocab, K, stat + row * splits + split, lists + (row * splits + split) * K);
}

// The same for BF16 rows that start on 16-byte boundaries, which stay packed: the maximum and the comparisons
// take two logits an instruction, as do the subtraction of the maximum, the multiplication by log2 e and the sum.
// The subtraction comes first: a slice whose every logit is masked by a large finite value has weights of 1.
template <int E>
__global__ void __launch_bounds__(kThreads)
    beam_slice_bf16_kernel(const bf16 *__restrict__ logits, int64_t ld, int vocab, int K, int splits,
                           Slice *__restrict__ stat, u64 *__restrict__ lists) {
    __shared__ TopShared sh;
    __shared__ float redm[kWarps], redk[kWarps];
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const int64_t row = blockIdx.x / splits;
    const int split = (int)(blockIdx.x % splits);
    const int base = split * (E * kThreads);
    const bf16 *src = logits + row * ld;
    uint32_t r[E / 2];
    auto index = [&](int e) { return base + (e / 8 * kThreads + (int)threadIdx.x) * 8 + e % 8; };
#pragma unroll
    for (int v = 0; v < E / 8; ++v) {
        const int i = index(8 * v);
        uint4 q = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);  // -inf
        if (i + 8 <= vocab) {
            q = *reinterpret_cast<const uint4 *>(src + i);
        } else if (i < vocab) {
            uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (i + u < vocab) {
                    const uint32_t bits = (uint32_t)__bfloat16_as_ushort(src[i + u]) << (u & 1 ? 16 : 0);
                    w[u / 2] = (w[u / 2] & (u & 1 ? 0xffffu : 0xffff0000u)) | bits;
                }
            q = make_uint4(w[0], w[1], w[2], w[3]);
        }
        r[4 * v] = q.x, r[4 * v + 1] = q.y, r[4 * v + 2] = q.z, r[4 * v + 3] = q.w;
    }
    auto two = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162 *>(&w); };
    __nv_bfloat162 top2 = two(r[0]);
#pragma unroll
    for (int i = 1; i < E / 2; ++i) top2 = __hmax2(top2, two(r[i]));
    const float mine = fmaxf(__low2float(top2), __high2float(top2));
    float m, bound;
    slice_bound(mine, K, redm, redk, m, bound, sh);
    float sum = 0.f;
    if (m > -INFINITY && m < INFINITY) {
        const u64 minus = pair(-m, -m), log2e = pair(1.4426950408889634f, 1.4426950408889634f);
        u64 total = 0;  // two zeros
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
            const float2 y = halves(mul2(add2(pair(__uint_as_float(r[i] << 16), __uint_as_float(r[i] & 0xffff0000u)), minus), log2e));
            total = add2(total, pair(exp2_ftz(y.x), exp2_ftz(y.y)));
        }
        const float2 t = halves(total);
        sum = t.x + t.y;
    } else if (m == -INFINITY) {  // all -inf, or NaN
#pragma unroll
        for (int i = 0; i < E / 2; ++i) sum += __hbeq2(two(r[i]), __bfloat162bfloat162(__float2bfloat16_rn(-INFINITY))) ? 0.f : NAN;
    } else {
        sum = NAN;
    }
    finish_slice<bf16>(warp_sum(sum), m, [&](auto &&use) {
        if (mine < bound) return;
        const __nv_bfloat162 b2 = __bfloat162bfloat162(__float2bfloat16_rn(bound));  // a logit: exact
#pragma unroll
        for (int v = 0; v < E / 8; ++v) {
            uint32_t hot = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) hot |= (__hge2_mask(two(r[4 * v + i]), b2) & 0x10001u) << i;  // bit i: low, 16 + i: high
            for (; hot; hot &= hot - 1) {
                const int e = __ffs(hot) - 1;
                use(index(8 * v) + 2 * (e & 15) + (e >> 4));
            }
        }
    }, sh, src, base, E * kThreads, vocab, K, stat + row * splits + split, lists + (row * splits + split) * K);
}

// ------------------------------------------------------------------- merging

// Largest value of the type below x (x finite).
template <typename T> __device__ __forceinline__ float next_below(float x);
template <> __device__ __forceinline__ float next_below<float>(float x) { return nextafterf(x, -INFINITY); }
template <> __device__ __forceinline__ float next_below<bf16>(float x) {
    if (x == 0.f) return -__uint_as_float(0x00010000u);
    const uint32_t u = __float_as_uint(x);
    return __uint_as_float(x > 0.f ? u - 0x10000u : u + 0x10000u);
}

struct Row {
    float score, max, logsum;
    int kind;  // 0: finite log-probabilities, 1: every candidate is -inf, 2: finished
};

// score + log softmax.  The maximum goes first: a row at the type's lowest value keeps its uniform weights.
__device__ __forceinline__ float candidate(const Row &r, float logit) {
    const float c = r.score + ((logit - r.max) - r.logsum);
    return c == c ? c : -INFINITY;  // NaN ranks as -inf
}

// One CTA per batch row: joins the rows' softmax sums and ranks each row's candidates by (value, lower flat
// index), a warp for a row, then ranks the rows' against one another by counting and writes the new beams.
// Latency is all it costs (about 5 us), so its start overlaps the slices' end.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    beam_merge_kernel(const T *__restrict__ logits, int64_t ld, const float *__restrict__ scores,
                      const uint8_t *__restrict__ finished, int64_t eos, int beams, int vocab, int splits, int stable,
                      const Slice *__restrict__ stat, const u64 *__restrict__ lists, float *__restrict__ out_scores,
                      int64_t *__restrict__ out_parents, int64_t *__restrict__ out_tokens,
                      uint8_t *__restrict__ out_finished) {
    __shared__ TopShared sh;
    __shared__ Row rows[kMaxBeams];
    __shared__ u64 lead[kMaxBeams][kMaxBeams];  // each row's K best candidates, in order
    __shared__ u64 kept[kMaxBeams];
    asm volatile("griddepcontrol.wait;\n" ::: "memory");  // the slices, as this launch may have begun before they ended
    const int64_t b = blockIdx.x;
    const int K = beams, tid = threadIdx.x, lane = tid & 31, per = splits * K;
    const unsigned all = 0xffffffffu;
    for (int w = tid >> 5; w < beams; w += kWarps) {  // a warp for each row
        const int64_t row = b * beams + w;
        const u64 *list = lists + row * per;
        u64 x = lane < per ? list[lane] : 0ull;  // on its way while the sums are joined
        Row r;
        r.score = scores[row];
        const bool done = finished && finished[row];
        float m = -INFINITY, s = 0.f;
        bool bad = false;
        for (int i = lane; i < splits; i += 32) {
            const Slice t = stat[row * splits + i];
            bad |= t.max != t.max;
            const float n = fmaxf(m, t.max);
            if (t.max > -INFINITY) s = s * (m > -INFINITY ? expf(m - n) : 0.f) + t.sum * expf(t.max - n);
            m = n;
        }
        bad = __any_sync(all, bad);
        float top = m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(all, top, o));
        s = warp_sum(m > -INFINITY ? s * expf(m - top) : 0.f);
        r.max = top;
        r.logsum = logf(s);
        r.kind = bad || top == -INFINITY || r.score != r.score || r.score == -INFINITY;
        if (done) r.kind = 2;
        const uint32_t flat = (uint32_t)w * (uint32_t)vocab;
        u64 best;
        if (r.kind == 0) {
            auto cand = [&](u64 y) { return y ? make_key(candidate(r, key_value(y)), flat + key_index(y)) : 0ull; };
            best = warp_sort_desc(cand(x));
            for (int i0 = 32; i0 < per; i0 += 32) {
                x = i0 + lane < per ? list[i0 + lane] : 0ull;
                const u64 y = __shfl_sync(all, warp_sort_desc(cand(x)), 31 - lane);
                best = warp_sort_desc(best > y ? best : y);
            }
        } else if (r.kind == 1) {  // every candidate is -inf: the lowest tokens
            best = lane < vocab ? make_key(-INFINITY, flat + lane) : 0ull;
        } else {  // finished: the end token keeps the score, then the lowest other tokens
            const int t = lane - 1 < (int)eos ? lane - 1 : lane;
            best = lane == 0 ? make_key(r.score == r.score ? r.score : -INFINITY, flat + (uint32_t)eos)
                             : (t < vocab ? make_key(-INFINITY, flat + t) : 0ull);
            best = warp_sort_desc(best);  // a score of -inf ties with them
        }
        if (lane < K) lead[w][lane] = best;
        if (lane == 0) rows[w] = r;
    }
    if (tid < K) kept[tid] = 0;
    __syncthreads();
    // a candidate's rank: the larger ones of every row, counted until it falls out
    for (int i = tid; i < beams * K; i += kThreads) {
        const int w = i / K, j = i % K;
        const u64 x = lead[w][j];
        int rank = x ? j : K;
        for (int v = 0; v < beams && rank < K; ++v)
            if (v != w)
                for (int q = 0; q < K && rank < K && lead[v][q] > x; ++q) ++rank;
        if (rank < K) kept[rank] = x;
    }
    __syncthreads();
    // Rounding may give unlisted logits (below the row's list) the value of a listed one and a lower index.
    // That can matter only where the row's last listed candidate reaches the selection and the type's next
    // value below its logit already rounds to the same candidate: such a row is read again, by candidate.
    const uint32_t kth = (uint32_t)(kept[K - 1] >> 32);
    const bool reach = tid < beams && vocab > K && rows[tid].kind == 0 && (uint32_t)(lead[tid][K - 1] >> 32) >= kth;
    if (__syncthreads_or(reach)) {
        for (int w = 0; w < beams; ++w) {
            const Row r = rows[w];
            if (r.kind != 0 || vocab <= K || (uint32_t)(lead[w][K - 1] >> 32) < kth) continue;
            u64 lowest = ~0ull;  // the row's K-th largest logit
            for (int k = 0; k < K; ++k) {
                u64 m = 0;
                for (int j = tid; j < per; j += kThreads) {
                    const u64 x = lists[(b * beams + w) * per + j];
                    if (x < lowest && x > m) m = x;
                }
                lowest = block_max(m, sh);
            }
            const float x = key_value(lowest);
            if (!(x > -INFINITY) || candidate(r, next_below<T>(x)) != candidate(r, x)) continue;
            // the row's K best by candidate, merged with the other rows' candidates kept so far
            const uint32_t flat = (uint32_t)w * (uint32_t)vocab;
            u64 last = ~0ull;
            u64 mine = 0;  // thread k < K: the row's k-th
            for (int k = 0; k < K; ++k) {
                u64 m = 0;
                for (int i = tid; i < vocab; i += kThreads) {
                    const u64 y = make_key(candidate(r, Elem<T>::to_float(logits[(b * beams + w) * ld + i])), flat + i);
                    if (y < last && y > m) m = y;
                }
                last = block_max(m, sh);
                if (tid == k) mine = last;
            }
            u64 other = tid < K ? kept[tid] : 0ull;
            if (other && key_index(other) / (uint32_t)vocab == (uint32_t)w) other = 0;  // its own are in `mine`
            __syncthreads();
            // 2 K distinct keys at most, in the first threads
            if (tid < K) {
                sh.list[tid] = mine;
                sh.list[K + tid] = other;
                kept[tid] = 0;
            }
            __syncthreads();
            if (tid < 2 * K && sh.list[tid]) {
                int rank = 0;
                for (int j = 0; j < 2 * K; ++j) rank += sh.list[j] > sh.list[tid];
                if (rank < K) kept[rank] = sh.list[tid];
            }
            __syncthreads();
        }
    }
    if (tid < 32) {
        const bool on = tid < K;
        const u64 x = on ? kept[tid] : 0ull;
        const uint32_t at = key_index(x);
        const int parent = on ? (int)(at / (uint32_t)vocab) : -1 - tid;
        const int64_t token = on ? at % (uint32_t)vocab : 0;
        int slot = tid;
        if (stable) {
            // the first child of a parent takes its slot, the others the free slots in turn
            const unsigned same = __match_any_sync(all, parent);
            const bool first = (same & ((1u << tid) - 1)) == 0;
            unsigned taken = on ? 1u << parent : 0u;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) taken |= __shfl_xor_sync(all, taken, o);
            const unsigned later = __ballot_sync(all, on && !first);
            if (on) {
                if (first) {
                    slot = parent;
                } else {
                    unsigned open = ~taken;
                    for (int n = __popc(later & ((1u << tid) - 1)); n > 0; --n) open &= open - 1;
                    slot = __ffs(open) - 1;
                }
            }
        }
        if (on) {
            const int64_t o = b * beams + slot;
            out_scores[o] = key_value(x);
            out_parents[o] = parent;
            out_tokens[o] = token;
            if (out_finished)
                out_finished[o] = (finished && finished[b * beams + parent]) || (eos >= 0 && token == eos);
        }
    }
}

// Logits per thread of the slice kernel and the splits of a row: as many as the registers hold (a CTA's fixed
// work is then least) where the rows alone fill the GPU, 8 (more CTAs per row) where they do not.
struct BeamPlan {
    int e, splits;
};
BeamPlan beam_plan(int64_t rows, int64_t vocab, bool packed) {
    BeamPlan p;
    p.e = packed ? 64 : 32;
    if (p.e == 64 && rows * ceil_div(vocab, 64 * kThreads) < 2 * kNumSMs) p.e = 32;
    if (p.e == 32 && rows * ceil_div(vocab, 32 * kThreads) < kNumSMs) p.e = 8;
    p.splits = (int)ceil_div(vocab, p.e * kThreads);
    return p;
}

template <typename T> using SliceFn = void (*)(const T *, int64_t, int, int, int, Slice *, u64 *);
SliceFn<float> slice_fn(const float *, bool vec, int e) {
    if (vec) return e == 32 ? beam_slice_kernel<float, 32, true> : beam_slice_kernel<float, 8, true>;
    return e == 32 ? beam_slice_kernel<float, 32, false> : beam_slice_kernel<float, 8, false>;
}
SliceFn<bf16> slice_fn(const bf16 *, bool vec, int e) {
    if (vec) return e == 64 ? beam_slice_bf16_kernel<64> : (e == 32 ? beam_slice_bf16_kernel<32> : beam_slice_bf16_kernel<8>);
    return e == 32 ? beam_slice_kernel<bf16, 32, false> : beam_slice_kernel<bf16, 8, false>;
}

// ------------------------------------------------------------------ reordering

constexpr int kMaxTensors = 32;
struct Tensors {
    void *base[kMaxTensors];
    int64_t stride[kMaxTensors];  // bytes between rows
    int64_t units[kMaxTensors];   // access units per row
    int64_t first[kMaxTensors + 1];  // first tile of each tensor
    int count;
};

constexpr int kUnroll = 4;  // columns a thread moves at a time

// In place: each thread owns columns of one group's rows and reads all of them that move before it writes
// any, so permutations and copies need no second buffer, and rows that stay cost nothing.  Bound by HBM: 16
// groups of 4 rows of 12.6 MB, half of them moved, take 132 us (127 at the copy rate), all of them 248 (254).
template <typename U, int W>
__global__ void __launch_bounds__(kThreads)
    reorder_rows_kernel(const Tensors t, const int64_t *__restrict__ parents, int beams, int64_t groups, int *status) {
    int k = 0;
    while (k + 1 < t.count && (int64_t)blockIdx.x >= t.first[k + 1]) ++k;
    const int64_t tile = blockIdx.x - t.first[k];
    const int64_t group = tile % groups, col0 = tile / groups * (kThreads * kUnroll) + threadIdx.x;
    int src[W];
    bool any = false;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        src[i] = i;
        if (i < beams) {
            const int64_t s = parents[group * beams + i];
            if (s >= 0 && s < beams)
                src[i] = (int)s;
            else if (status && threadIdx.x == 0)
                *(volatile int *)status = 0x8;  // the row keeps its state
            any |= src[i] != i;
        }
    }
    if (!any) return;
    char *base = static_cast<char *>(t.base[k]) + group * beams * t.stride[k];
    const int64_t stride = t.stride[k], units = t.units[k];
    constexpr int kAt = W <= 4 ? kUnroll : (W <= 8 ? 2 : 1);  // columns in registers at a time
#pragma unroll
    for (int u0 = 0; u0 < kUnroll; u0 += kAt) {
        U x[kAt][W];
#pragma unroll
        for (int u = 0; u < kAt; ++u)
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (src[i] != i && col0 + (u0 + u) * kThreads < units)
                    x[u][i] = *(reinterpret_cast<const U *>(base + src[i] * stride) + col0 + (u0 + u) * kThreads);
#pragma unroll
        for (int u = 0; u < kAt; ++u)
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (src[i] != i && col0 + (u0 + u) * kThreads < units)
                    *(reinterpret_cast<U *>(base + i * stride) + col0 + (u0 + u) * kThreads) = x[u][i];
    }
}

// The same for more than 16 beams, whose columns would take all of a thread's registers: the rows that move pass
// through shared memory, 1 KB of each at a time (2 groups of 32 rows of 12.6 MB, half of them moved: 156 to 171 us, from
// registers 217; 4 groups of 16: 178, from registers in 8-byte columns 133).
constexpr int kTileUnits = 64;
__global__ void __launch_bounds__(kThreads)
    reorder_tiles_kernel(const Tensors t, const int64_t *__restrict__ parents, int beams, int64_t groups, int *status) {
    __shared__ uint4 tile[kMaxBeams][kTileUnits];
    __shared__ int src[kMaxBeams];
    int k = 0;
    while (k + 1 < t.count && (int64_t)blockIdx.x >= t.first[k + 1]) ++k;
    const int64_t at = blockIdx.x - t.first[k];
    const int64_t group = at % groups, unit = at / groups * kTileUnits + threadIdx.x % kTileUnits;
    if (threadIdx.x < beams) {
        const int64_t s = parents[group * beams + threadIdx.x];
        const bool in = s >= 0 && s < beams;
        src[threadIdx.x] = in ? (int)s : (int)threadIdx.x;
        if (!in && status) *(volatile int *)status = 0x8;  // the row keeps its state
    }
    __syncthreads();
    char *base = static_cast<char *>(t.base[k]) + group * beams * t.stride[k] + unit * 16;
    const int64_t stride = t.stride[k];
    constexpr int kStep = kThreads / kTileUnits;
    const int row = threadIdx.x / kTileUnits, u = threadIdx.x % kTileUnits;
    if (unit < t.units[k])
#pragma unroll 8
        for (int i = row; i < beams; i += kStep)
            if (src[i] != i) tile[i][u] = *reinterpret_cast<const uint4 *>(base + src[i] * stride);
    __syncthreads();
    if (unit < t.units[k])
#pragma unroll 8
        for (int i = row; i < beams; i += kStep)
            if (src[i] != i) *reinterpret_cast<uint4 *>(base + i * stride) = tile[i][u];
}

template <typename U>
int reorder_launch(Tensors t, const int64_t *row_bytes, const int64_t *parents, int64_t groups, int beams, int *status,
                   cudaStream_t st) {
    const bool tiled = sizeof(U) == 16 && beams > 16;
    int64_t tiles = 0;
    for (int i = 0; i < t.count; ++i) {
        t.units[i] = row_bytes[i] / (int64_t)sizeof(U);
        t.first[i] = tiles;
        tiles += groups * ceil_div(t.units[i], tiled ? kTileUnits : kThreads * kUnroll);
    }
    t.first[t.count] = tiles;
    if (tiles > 0x7fffffff) return BDM_ERR_UNSUPPORTED;
    if (tiles == 0) return BDM_OK;
    const unsigned grid = (unsigned)tiles;
    if (tiled)
        reorder_tiles_kernel<<<grid, kThreads, 0, st>>>(t, parents, beams, groups, status);
    else if (beams <= 4)
        reorder_rows_kernel<U, 4><<<grid, kThreads, 0, st>>>(t, parents, beams, groups, status);
    else if (beams <= 8)
        reorder_rows_kernel<U, 8><<<grid, kThreads, 0, st>>>(t, parents, beams, groups, status);
    else if constexpr (sizeof(U) < 16) {
        if (beams <= 16)
            reorder_rows_kernel<U, 16><<<grid, kThreads, 0, st>>>(t, parents, beams, groups, status);
        else if constexpr (sizeof(U) < 8)
            reorder_rows_kernel<U, 32><<<grid, kThreads, 0, st>>>(t, parents, beams, groups, status);
    }
    return launch_status();
}

}  // namespace
}  // namespace bdm

extern "C" int64_t bdm_beam_select_workspace_bytes(int64_t batch, int beams, int64_t vocab) {
    using namespace bdm;
    if (batch < 0 || beams <= 0 || vocab <= 0 || beams > kMaxBeams || vocab > kMaxVocab ||
        vocab * beams >= 0xffffffffll)
        return -1;
    const BeamPlan p = beam_plan(batch * beams, vocab, false);  // never fewer splits than the packed plan's
    return batch * beams * p.splits * ((int64_t)beams * 8 + 8);
}

extern "C" int bdm_beam_select(const void *logits, int64_t ld, int64_t batch, int beams, int64_t vocab, int dtype,
                               const float *scores, const uint8_t *finished, int64_t eos_token, int stable_slots,
                               float *out_scores, int64_t *out_parents, int64_t *out_tokens, uint8_t *out_finished,
                               void *workspace, int64_t workspace_bytes, void *stream) {
    using namespace bdm;
    if (batch < 0 || beams <= 0 || vocab <= 0 || ld < 0 || eos_token < -1 || eos_token >= vocab) return BDM_ERR_INVALID;
    if (finished && eos_token < 0) return BDM_ERR_INVALID;
    if (!valid_dtype(dtype)) return BDM_ERR_DTYPE;
    if (beams > kMaxBeams || vocab > kMaxVocab || vocab * beams >= 0xffffffffll) return BDM_ERR_UNSUPPORTED;
    if (batch == 0) return BDM_OK;
    if (!logits || !scores || !out_scores || !out_parents || !out_tokens) return BDM_ERR_INVALID;
    const int64_t rows = batch * beams;
    const bool vec = (reinterpret_cast<uintptr_t>(logits) & 15) == 0 && (ld * (dtype == BDM_BF16 ? 2 : 4)) % 16 == 0;
    const BeamPlan p = beam_plan(rows, vocab, vec && dtype == BDM_BF16);
    if (!workspace || workspace_bytes < bdm_beam_select_workspace_bytes(batch, beams, vocab)) return BDM_ERR_WORKSPACE;
    if (rows * p.splits > 0x7fffffff) return BDM_ERR_UNSUPPORTED;
    cudaStream_t st = as_stream(stream);
    u64 *lists = static_cast<u64 *>(workspace);
    Slice *stat = reinterpret_cast<Slice *>(lists + rows * p.splits * beams);
    const unsigned grid = (unsigned)(rows * p.splits);
    BDM_DISPATCH_DTYPE(dtype, T, {
        const T *x = static_cast<const T *>(logits);
        const SliceFn<T> slice = slice_fn(x, vec, p.e);
        slice<<<grid, kThreads, 0, st>>>(x, ld, (int)vocab, beams, p.splits, stat, lists);
        if (int rc = launch_status()) return rc;
        // a programmatic dependent launch: its start overlaps the slices' end
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)batch);
        cfg.blockDim = dim3(kThreads);
        cfg.stream = st;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        if (int rc = cuda_status(cudaLaunchKernelEx(&cfg, beam_merge_kernel<T>, x, ld, scores, finished, eos_token, beams,
                                                    (int)vocab, p.splits, stable_slots, (const Slice *)stat,
                                                    (const u64 *)lists, out_scores, out_parents, out_tokens, out_finished)))
            return rc;
    });
    return launch_status();
}

extern "C" int bdm_reorder_rows(void *const *bases, const int64_t *row_strides, const int64_t *row_bytes, int count,
                                const int64_t *parents, int64_t groups, int beams, int *status, void *stream) {
    using namespace bdm;
    if (count < 0 || groups < 0 || beams <= 0) return BDM_ERR_INVALID;
    if (beams > kMaxBeams) return BDM_ERR_UNSUPPORTED;
    if (count == 0 || groups == 0) return BDM_OK;
    if (!bases || !row_strides || !row_bytes || !parents) return BDM_ERR_INVALID;
    for (int i = 0; i < count; ++i)
        if (row_bytes[i] < 0 || row_strides[i] < row_bytes[i] || (row_bytes[i] && !bases[i])) return BDM_ERR_INVALID;
    cudaStream_t st = as_stream(stream);
    for (int width : {16, 8, 4, 1}) {  // the access that a tensor's rows allow
        Tensors t{};
        int64_t bytes[kMaxTensors];
        auto flush = [&]() {
            const int rc = t.count == 0 ? BDM_OK
                           : width == 16 ? reorder_launch<uint4>(t, bytes, parents, groups, beams, status, st)
                           : width == 8  ? reorder_launch<uint2>(t, bytes, parents, groups, beams, status, st)
                           : width == 4  ? reorder_launch<uint32_t>(t, bytes, parents, groups, beams, status, st)
                                         : reorder_launch<uint8_t>(t, bytes, parents, groups, beams, status, st);
            t.count = 0;
            return rc;
        };
        for (int i = 0; i < count; ++i) {
            const uint64_t bits = reinterpret_cast<uintptr_t>(bases[i]) | (uint64_t)row_strides[i] | (uint64_t)row_bytes[i];
            // 16 bytes, but 8 where the registers are to hold 9 to 16 rows' columns; tensors of odd sizes 4 or 1
            const int fits = bits % 16 == 0 ? (beams > 8 && beams <= 16 ? 8 : 16) : (bits % 4 == 0 ? 4 : 1);
            if (fits != width || row_bytes[i] == 0) continue;
            t.base[t.count] = bases[i];
            t.stride[t.count] = row_strides[i];
            bytes[t.count++] = row_bytes[i];
            if (t.count == kMaxTensors)
                if (int rc = flush()) return rc;
        }
        if (int rc = flush()) return rc;
    }
    return BDM_OK;
}
