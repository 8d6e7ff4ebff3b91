// Decay attention on the tensor cores: tensor maps, segments and launches (the kernel is in decay_walk_tc.cuh).
#include "decay_walk_tc.cuh"

namespace bdm {
namespace {

using namespace walk;

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
        if (w.width_c % 8) return false;
        if ((w.batch > 1 && !w.out_stride[0]) || (w.heads > 1 && !w.out_stride[2])) return false;
    }
    return encode_tiled() != nullptr;
}

// Segments of the time axis, and CTAs to a row's value columns: the split that makes the launches shortest, in
// units of a chunk of the main walk (1.7 us).  A CTA has an SM to itself; its start and end cost about three
// chunks, a chunk of half the columns 0.75, one of the state launch 0.6 of the walk's, the prefix launch and the
// dependent starts about six in all.  (8 x 4096 tokens x 8 heads of 128 with the state: two segments 103 us, two
// halves of the columns 83; halves also read a and b twice, but from L2.)
WalkSplit decay_walk_tc_split(int64_t rows, int64_t chunks, int width_c, int sms) {
    WalkSplit best{1, (int)chunks, 1, (int)chunks, 1};
    double cost = (double)ceil_div(rows, sms) * (chunks + 3.0);
    for (int v = 1; v <= (width_c > 64 ? 2 : 1); ++v) {
        const double chunk = v == 2 ? 0.75 : 1.0;
        const int64_t r = rows * v;
        for (int64_t s = 1; s <= chunks / 4 + 1 && s <= 128 && r * (s - 1) < 2 * sms; ++s) {
            const int64_t c0 = ceil_div(chunks, s);
            int64_t u = s > 1 ? sms / (r * (s - 1)) : 1;
            if (u > c0 / 2) u = c0 / 2;
            if (u < 1) u = 1;
            const int64_t sc = ceil_div(c0, u), c = sc * u, n = ceil_div(chunks, c);
            if (s > 1 && n < 2) continue;
            double t = ceil_div(r * n, sms) * (chunk * c + 3.0);
            if (n > 1) t += ceil_div(r * (n - 1) * u, sms) * (0.6 * chunk * sc + 3.0) + 6.0;
            if (t < cost) cost = t, best = WalkSplit{(int)n, (int)c, (int)u, (int)sc, v};
        }
    }
    return best;
}

int decay_walk_tc_launch(const bdm_decay_walk_args &w, Params p, const WalkSplit &split, void *workspace, cudaStream_t st) {
    EncodeTiled fn = encode_tiled();
    if (!fn) return BDM_ERR_UNSUPPORTED;
    TcParams tp{};
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
    p.seg = static_cast<float *>(workspace);
    tp.p = p;
    tp.sub = split.sub;
    tp.scps = split.scps;
    tp.vsplit = split.vsplit;
    tp.z = p.seg + p.batch * p.heads * p.nseg * (int64_t)p.wab * p.wc;
    // ragged rows in more than one wave (24 x 1333, 192 CTAs: 62 us in the order of the batch, 43 us sorted); a
    // CTA's sort is a loop over the batch, so large batches, whose many waves level out by themselves, go without
    tp.longest_first = p.lengths && p.batch > 1 && p.batch <= 256 && p.batch * p.heads * p.nseg * split.vsplit > kNumSMs;
    const int terms = p.state_out ? 3 : 2;
    const bool wide = p.wc > 64 && split.vsplit == 1;
    auto run = p.wab > 64 ? (wide ? tc_launch_22 : tc_launch_21) : (wide ? tc_launch_12 : tc_launch_11);
    if (p.nseg > 1) {
        if (int rc = run(tp, maps, kTcState, terms, false, st)) return rc;
        if (int rc = decay_prefix_launch(p, tp.z, split.sub, split.scps, st)) return rc;
    }
    return run(tp, maps, w.out_dtype == BDM_F32 ? kTcFloat : kTcBf16, terms, p.nseg > 1 || w.overlap, st);
}

}  // namespace bdm
