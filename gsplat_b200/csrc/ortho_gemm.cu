// Tensor maps and the choice of a tile for the products of ortho_gemm.cuh.
#include "ortho_gemm.cuh"
#include "ortho_gemm_pair.cuh"

namespace gsb {

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                              const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeFn encode_fn() {
    static const EncodeFn fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeFn>(f);
    }();
    return fn;
}

// A batch of [rows, cols] planes read in boxes of 64 columns x `box_rows`; zeros outside.
static bool encode(CUtensorMap *map, const __half *base, const OrthoPlanes &p, int rows, int cols, long long batch,
                   int box_rows) {
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)batch};
    const cuuint64_t strides[2] = {(cuuint64_t)p.ld * 2, (cuuint64_t)p.stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, ones[3] = {1, 1, 1};
    return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half *>(base), dims, strides, box, ones,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int sm_count() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    return sms;
}

OrthoTile ortho_tile(const OrthoGemm &g, int sms) {
    // The tile with the least time: rounds over the SMs x cycles of a product 16 deep / blocks that share the depth. The
    // cycles are measured: the operand bytes that an SM's shared memory delivers bound them where few SMs work, those
    // that the L2 delivers (5 to 6.3 KB a cycle with all of them) where all do. A 128 x 64 tile 79, or 122 for hi planes alone on all SMs;
    // 128 x 128 112 split, 126 or 162; a pair's 256 x 256 165 split (also where few work, for its longer end), 237.
    const int tm = (g.M + kBM - 1) / kBM, tn = (g.N + 127) / 128, tn64 = (g.N + 63) / 64;
    const int pm = (g.M + kPair - 1) / kPair, pn = (g.N + kPair - 1) / kPair;
    const long long n64 = g.batch * (g.symmetric ? tm * (tm + 1) - (2 * tm - tn64) : tm * tn64);
    const long long n128 = g.batch * (g.symmetric ? tm * (tm + 1) / 2 : tm * tn);
    const long long n256 = g.batch * (g.symmetric ? pm * (pm + 1) / 2 : pm * pn);
    const int r64 = g.split ? tile_ranks<true, 64>(g, n64, sms) : tile_ranks<false, 64>(g, n64, sms);
    const int r128 = g.split ? tile_ranks<true, 128>(g, n128, sms) : tile_ranks<false, 128>(g, n128, sms);
    const long long t64 = (n64 + sms - 1) / sms * (g.split || n64 * r64 <= sms / 2 ? 79 : 122) / r64;
    const long long t128 = (n128 + sms - 1) / sms * (g.split ? 112 : n128 * r128 <= sms / 2 ? 126 : 162) / r128;
    const long long t256 = (n256 + sms / 2 - 1) / (sms / 2) * (g.split || n256 <= sms / 4 ? 165 : 237);
    if (t256 < t128 && t256 < t64 && (g.split || g.K <= kHiDepth)) return {256, 1};
    return t64 < t128 ? OrthoTile{64, r64} : OrthoTile{128, r128};
}

int ortho_gemm(const OrthoGemm &g, const MuonTable *table, cudaStream_t stream) {
    if (encode_fn() == nullptr) return set_error(kErrUnsupported, "orthogonalize: the driver offers no tensor maps");
    GemmMaps maps;
    const int sms = sm_count(), columns = ortho_tile(g, sms).columns, bn = std::min(columns, 128);
    for (int i = 0; i < g.pairs; ++i) {
        const int qr = g.q_k_major ? g.N : g.K, qc = g.q_k_major ? g.K : g.N, qb = g.q_k_major ? bn : 64;
        if (!encode(&maps.p_hi[i], g.p[i].hi, g.p[i], g.M, g.K, g.batch, kBM) ||
            !encode(&maps.p_lo[i], g.p[i].lo, g.p[i], g.M, g.K, g.batch, kBM) ||
            !encode(&maps.q_hi[i], g.q[i].hi, g.q[i], qr, qc, g.batch, qb) ||
            !encode(&maps.q_lo[i], g.q[i].lo, g.q[i], qr, qc, g.batch, qb))
            return set_error(kErrLaunch, "orthogonalize: a tensor map of %d x %d could not be made", qr, qc);
    }
    if (g.pairs == 1) {
        maps.p_hi[1] = maps.p_hi[0];
        maps.p_lo[1] = maps.p_lo[0];
        maps.q_hi[1] = maps.q_hi[0];
        maps.q_lo[1] = maps.q_lo[0];
    }
    static const MuonTable none = {};
    const MuonTable &tab = table ? *table : none;
    if (columns == 256) {
        const int e = g.split ? ortho_pair_launch<true>(g, maps, tab, sms, stream) : ortho_pair_launch<false>(g, maps, tab, sms, stream);
        if (e != kPairUnfit) return e; // else 128 x 128 tiles, whose tensor maps are the same
    }
    if (bn == 64)
        return g.split ? ortho_gemm_launch<true, 64>(g, maps, tab, sms, stream) : ortho_gemm_launch<false, 64>(g, maps, tab, sms, stream);
    return g.split ? ortho_gemm_launch<true, 128>(g, maps, tab, sms, stream) : ortho_gemm_launch<false, 128>(g, maps, tab, sms, stream);
}

} // namespace gsb
