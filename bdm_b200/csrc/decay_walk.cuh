// Shared pieces of the decay-attention walk: parameters, the segmentation of the time axis, and the
// state a segment starts from.
//
// Walk (per batch row and head, lam = exp(log_decay)), n valid tokens:
//   forward:  out_t = scale * (sum_{s<=t} lam^(t-s) (a_t.b_s) c_s + lam^(t+1)   a_t X)
//             Y     = lam^n X + sum_s lam^(n-1-s) b_s c_s^T
//   reverse:  out_t = scale * (sum_{s>=t} lam^(s-t) (a_t.b_s) c_s + lam^(n-1-t) a_t X)
//             Y     = lam^n X + sum_s lam^(s+1)   b_s c_s^T
// X = state_in * state_in_mul, state_out = Y * state_out_mul.  o = forward(q, k, v); the gradients are
// the same walk: dq = forward(do, v, k), dk = reverse(v, do, q), dv = reverse(k, q, do).
//
// In a chunk of kChunk tokens starting at t0, row r = t - t0 of n' = min(kChunk, n - t0) valid ones, the
// exponents are: inside t-s (or s-t); reading the carried state r+1 (n'-1-r); writing it n'-1-r (r+1);
// carrying it n'.  The time axis is cut into segments of whole chunks when there are too few (row, head)
// pairs for the SMs: a first launch leaves the segments' own states (X = 0) in the workspace, a second sums
// what each segment starts from (in order: no atomics), and the main launch walks all segments side by side.
#pragma once

#include "common.cuh"

namespace bdm {
namespace walk {

constexpr int kChunk = 64;
constexpr int kMaxWidth = 128;  // of a, b and of c: what one CTA's tiles hold
// Below this log-decay a power is zero in FP32 from the first token on; clamping keeps 0 * -inf away.
constexpr float kLogFloor = -1.0e4f;

struct Params {
    const void *a, *b, *c;
    int64_t as[3], bs[3], cs[3], os[3];  // strides of batch, token, head (elements)
    int ag, bg, cg;                      // heads sharing one head of a, b, c
    void *out;
    const float *log_decay;
    const int64_t *lengths;
    const float *state_in;
    float *state_out;
    float in_mul, out_mul;
    int in_t, out_t;  // state stored [wc, wab] instead of [wab, wc]
    float *seg;       // what each segment starts from, beside the given state: [batch*heads, nseg, wab * wc]
    int64_t batch, time;
    int heads, wab, wc, reverse;
    float scale;
    int nseg, cps;  // segments, chunks per segment
    int *status;
};

__device__ __forceinline__ float head_log_decay(const Params &p, int h) {
    const float g = p.log_decay[h];
    return g < kLogFloor ? kLogFloor : g;
}
__device__ __forceinline__ int64_t row_tokens(const Params &p, int64_t b) {
    if (!p.lengths) return p.time;
    const int64_t n = p.lengths[b];
    return n < 0 ? 0 : (n > p.time ? p.time : n);
}

// One segment of one row: its chunks [c0, c1), the row's chunks, and its place in the walk.
struct Span {
    int64_t n, c0, c1, chunks;
    bool last;  // the walk ends here: this segment writes the final state
};
__device__ __forceinline__ Span span_of(const Params &p, int64_t n, int seg) {
    Span s;
    s.n = n;
    s.chunks = (n + kChunk - 1) / kChunk;
    s.c0 = (int64_t)seg * p.cps;
    s.c1 = s.c0 + p.cps;
    if (s.c0 > s.chunks) s.c0 = s.chunks;
    if (s.c1 > s.chunks) s.c1 = s.chunks;
    if (p.reverse || s.chunks == 0)
        s.last = seg == 0;
    else
        s.last = s.c1 == s.chunks && s.c0 < s.c1;
    return s;
}

}  // namespace walk

// How a walk is cut up: segments of a row and their chunks, sub-segments of one in the state launch and theirs,
// CTAs that share a row's value columns.
struct WalkSplit {
    int nseg, cps, sub, scps, vsplit;
};

// Sums the segments' start states from z, [batch*heads, (nseg - 1) * sub, wab * wc], the own states of the
// sub-segments (scps chunks each, sub in a segment) of all segments but the last one walked.
int decay_prefix_launch(const walk::Params &p, const float *z, int sub, int scps, cudaStream_t st);

// The tensor-core walk (decay_walk_tc.cu): BF16 operands that TMA can address.
bool decay_walk_tc_takes(const bdm_decay_walk_args &w);
WalkSplit decay_walk_tc_split(int64_t rows, int64_t chunks, int width_c, int sms);
int decay_walk_tc_launch(const bdm_decay_walk_args &w, walk::Params p, const WalkSplit &split, void *workspace,
                         cudaStream_t st);

}  // namespace bdm
