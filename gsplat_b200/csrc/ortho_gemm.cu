// Batched products of the Newton-Schulz iteration with their element-wise ends:
// one thread block a 64 x 64 tile of the result, 32-bit FMAs.
#include "ortho.cuh"

namespace gsb {

constexpr int kTile = 64, kDepth = 16, kGemmThreads = 256;

__device__ __forceinline__ float plane_at(const OrthoPlanes &p, long long b, int i, int j, bool lo) {
    const size_t at = (size_t)b * p.stride + (size_t)i * p.ld + j;
    float v = __half2float(p.hi[at]);
    if (lo) v += __half2float(p.lo[at]);
    return v;
}
__device__ __forceinline__ void plane_put(const OrthoPlanes &p, long long b, int i, int j, float v, bool lo) {
    const size_t at = (size_t)b * p.stride + (size_t)i * p.ld + j;
    const __half h = __float2half_rn(v);
    p.hi[at] = h;
    if (lo) p.lo[at] = __float2half_rn(v - __half2float(h));
}

// The epilogue of element (i, j); `mirror`: also at (j, i).
__device__ __forceinline__ void emit(const OrthoGemm &g, const MuonTable &tab, long long b, int i, int j, float acc,
                                     bool mirror) {
    const float *d = g.diag_in + (size_t)b * g.M;
    float v;
    switch (g.epilogue) {
    case kEpiGram:
        v = i == j ? 0.f : g.c[0] * acc;
        if (i == j) g.diag_out[(size_t)b * g.M + i] = g.c[1] * acc;
        break;
    case kEpiSquare:
        if (i == j) {
            g.diag_out[(size_t)b * g.M + i] = fmaf(g.c[3], d[i], fmaf(g.c[4] * d[i], d[i], g.c[5] * acc));
            v = 0.f;
        } else {
            v = fmaf(fmaf(g.c[1], d[i] + d[j], g.c[0]), plane_at(g.e, b, i, j, g.split), g.c[2] * acc);
        }
        break;
    case kEpiSym: v = g.c[0] * acc; break;
    case kEpiAnti: v = fmaf(fmaf(g.c[1], d[i] + d[j], g.c[0]), plane_at(g.e, b, i, j, true), g.c[2] * acc); break;
    default: v = fmaf(g.c[0] + d[i], plane_at(g.e, b, i, j, true), g.c[1] * acc) * g.c[2];
    }
    const size_t at = g.transposed ? (size_t)j * g.M + i : (size_t)i * g.N + j;
    if (g.epilogue == kEpiOut) {
        store_from_f32(g.y, (size_t)b * g.M * g.N + at, g.dtype, v);
    } else if (g.epilogue == kEpiMuon) {
        const int t = muon_tensor_of(tab, b);
        const size_t o = (size_t)(b - tab.first[t]) * g.M * g.N + at;
        store_from_f32(tab.param[t], o, tab.dtype,
                       muon_param(load_as_f32(tab.param[t], o, tab.dtype), v, tab.lr[t], tab.decay[t]));
    } else {
        const bool lo = g.split || g.epilogue == kEpiApply;
        plane_put(g.out, b, i, j, v, lo);
        if (mirror) plane_put(g.out, b, j, i, v, lo);
    }
}

__global__ void __launch_bounds__(kGemmThreads)
    ortho_gemm_kernel(const __grid_constant__ OrthoGemm g, const __grid_constant__ MuonTable tab, int tiles_m, int tiles_n) {
    __shared__ float sp[kDepth][kTile + 1], sq[kDepth][kTile + 1];
    const long long b = blockIdx.x / ((long long)tiles_m * tiles_n);
    const int t = (int)(blockIdx.x % ((long long)tiles_m * tiles_n));
    const int ti = t / tiles_n, tj = t % tiles_n;
    if (g.symmetric && tj > ti) return;
    if (tab.n > 0 && !muon_visible(tab, muon_tensor_of(tab, b), b)) return;
    const int i0 = ti * kTile, j0 = tj * kTile;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {};
    for (int pair = 0; pair < g.pairs; ++pair)
        for (int k0 = 0; k0 < g.K; k0 += kDepth) {
            for (int e = threadIdx.x; e < kTile * kDepth; e += kGemmThreads) {
                const int r = e / kDepth, k = e % kDepth;
                sp[k][r] = i0 + r < g.M && k0 + k < g.K ? plane_at(g.p[pair], b, i0 + r, k0 + k, g.split) : 0.f;
                if (g.q_k_major) {
                    sq[k][r] = j0 + r < g.N && k0 + k < g.K ? plane_at(g.q[pair], b, j0 + r, k0 + k, g.split) : 0.f;
                } else {
                    const int kk = e / kTile, c = e % kTile;
                    sq[kk][c] = j0 + c < g.N && k0 + kk < g.K ? plane_at(g.q[pair], b, k0 + kk, j0 + c, g.split) : 0.f;
                }
            }
            __syncthreads();
            for (int k = 0; k < kDepth; ++k)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[r][c] = fmaf(sp[k][ty + 16 * r], sq[k][tx + 16 * c], acc[r][c]);
            __syncthreads();
        }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int i = i0 + ty + 16 * r, j = j0 + tx + 16 * c;
            if (i < g.M && j < g.N) emit(g, tab, b, i, j, acc[r][c], g.symmetric && ti != tj);
        }
}

int ortho_gemm(const OrthoGemm &g, const MuonTable *table, cudaStream_t stream) {
    const int tm = (g.M + kTile - 1) / kTile, tn = (g.N + kTile - 1) / kTile;
    const long long blocks = g.batch * tm * tn;
    if (blocks > 0x7fffffffll) return set_error(kErrInvalidArgument, "orthogonalize: too many tiles");
    static const MuonTable none = {};
    ortho_gemm_kernel<<<(unsigned)blocks, kGemmThreads, 0, stream>>>(g, table ? *table : none, tm, tn);
    return check_launch("ortho_gemm_kernel");
}

} // namespace gsb
