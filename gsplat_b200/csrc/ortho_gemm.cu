// Batched products of the Newton-Schulz iteration with their element-wise ends, on
// the fifth-generation tensor cores: one persistent block an SM, TMA into 128-byte-swizzled
// stages, tcgen05.mma into double-buffered TMEM accumulators, and eight warps that
// finish a tile while the next one is multiplied.
//
// A tile is 128 x 128 of the result, 64 deep a stage. With `split`, a stage holds
// the hi and lo planes of both operands and feeds three products (hi hi, hi lo, lo hi);
// the sum is taken out of the tensor cores every kChunk stages and continued in
// registers, since their 32-bit adder truncates and the bias of a long sum of
// squares would be seen in the diagonal of A.
#include <cuda.h>

#include "ortho.cuh"
#include "tcgen05.cuh"

namespace gsb {

constexpr int kBM = 128, kBN = 128, kBK = 64;
constexpr int kPlaneBytes = kBM * kBK * 2; // of one operand plane of a stage
constexpr int kSplitStages = 3, kHalfStages = 6;
constexpr int kChunk = 8;          // stages between two readings of the accumulator, split
constexpr int kEpilogueWarps = 8;  // four lane quarters x two column halves
constexpr int kGemmThreads = 32 * (kEpilogueWarps + 2);
constexpr int kTmemColumns = 2 * kBN;

struct GemmMaps {
    CUtensorMap p_hi[2], p_lo[2], q_hi[2], q_lo[2];
};

struct GemmShared {
    alignas(8) unsigned long long full[kHalfStages], empty[kHalfStages];
    unsigned long long acc_full[2], acc_empty[2];
    uint32_t tmem;
    int abort;
};

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, int x, int y, int z,
                                         unsigned long long *bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
                 : "memory");
}

// Eight values of a row of planes; past the row's 8-column groups, zeros.
__device__ __forceinline__ void load8(const OrthoPlanes &p, size_t at, bool lo, float v[8]) {
    const uint4 h = *reinterpret_cast<const uint4 *>(p.hi + at);
    const __half2 *hh = reinterpret_cast<const __half2 *>(&h);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(hh[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
    if (lo) {
        const uint4 l = *reinterpret_cast<const uint4 *>(p.lo + at);
        const __half2 *ll = reinterpret_cast<const __half2 *>(&l);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(ll[i]);
            v[2 * i] += f.x;
            v[2 * i + 1] += f.y;
        }
    }
}
__device__ __forceinline__ void store8(const OrthoPlanes &p, size_t at, bool lo, const float v[8]) {
    uint4 h, l;
    __half2 *hh = reinterpret_cast<__half2 *>(&h), *ll = reinterpret_cast<__half2 *>(&l);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        hh[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        const float2 f = __half22float2(hh[i]);
        ll[i] = __floats2half2_rn(v[2 * i] - f.x, v[2 * i + 1] - f.y);
    }
    *reinterpret_cast<uint4 *>(p.hi + at) = h;
    if (lo) *reinterpret_cast<uint4 *>(p.lo + at) = l;
}

// The epilogue of 32 columns from j of row i (i < M, j < N).
__device__ __forceinline__ void finish32(const OrthoGemm &g, const MuonTable &tab, int tensor, long long b, int i, int j,
                                         bool mirror, bool poisoned, float v[32]) {
    const float *d = g.diag_in + (size_t)b * g.M;
    const size_t erow = (size_t)b * g.e.stride + (size_t)i * g.e.ld;
    float di = 0.f;
    if (g.epilogue != kEpiGram && g.epilogue != kEpiSym) di = d[i];
#pragma unroll
    for (int c = 0; c < 32; c += 8) {
        if (j + c >= g.N) break;
        float *w = v + c;
        float e[8];
        switch (g.epilogue) {
        case kEpiGram:
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (i == j + c + k) {
                    g.diag_out[(size_t)b * g.M + i] = g.c[1] * w[k];
                    w[k] = 0.f;
                } else {
                    w[k] *= g.c[0];
                }
            }
            break;
        case kEpiSym:
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] *= g.c[0];
            break;
        case kEpiSquare:
        case kEpiAnti:
            load8(g.e, erow + j + c, g.split, e);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int jj = j + c + k;
                if (g.epilogue == kEpiSquare && i == jj) {
                    g.diag_out[(size_t)b * g.M + i] = fmaf(g.c[3], di, fmaf(g.c[4] * di, di, g.c[5] * w[k]));
                    w[k] = 0.f;
                } else {
                    w[k] = fmaf(fmaf(g.c[1], di + (jj < g.N ? d[jj] : 0.f), g.c[0]), e[k], g.c[2] * w[k]);
                }
            }
            break;
        default:
            load8(g.e, erow + j + c, true, e);
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] = fmaf(g.c[0] + di, e[k], g.c[1] * w[k]) * g.c[2];
        }
        if (g.epilogue == kEpiOut || g.epilogue == kEpiMuon) {
            const size_t base = (size_t)(b - (g.epilogue == kEpiMuon ? tab.first[tensor] : 0)) * g.M * g.N;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int jj = j + c + k;
                if (jj >= g.N) break;
                const float r = poisoned ? NAN : w[k];
                const size_t at = base + (g.transposed ? (size_t)jj * g.M + i : (size_t)i * g.N + jj);
                if (g.epilogue == kEpiOut)
                    store_from_f32(g.y, at, g.dtype, r);
                else
                    store_from_f32(tab.param[tensor], at, tab.dtype,
                                   muon_param(load_as_f32(tab.param[tensor], at, tab.dtype), r, tab.lr[tensor],
                                              tab.decay[tensor]));
            }
        } else {
            const bool lo = g.split || g.epilogue == kEpiApply;
            store8(g.out, (size_t)b * g.out.stride + (size_t)i * g.out.ld + j + c, lo, w);
            if (mirror) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (j + c + k >= g.N) break;
                    const size_t at = (size_t)b * g.out.stride + (size_t)(j + c + k) * g.out.ld + i;
                    const __half h = __float2half_rn(w[k]);
                    g.out.hi[at] = h;
                    if (lo) g.out.lo[at] = __float2half_rn(w[k] - __half2float(h));
                }
            }
        }
    }
}

struct TileAt {
    long long b;
    int i, j; // in tiles
};
// Tile t of the launch; symmetric results list the lower triangle by rows.
__device__ __forceinline__ TileAt tile_at(long long t, int per, int tiles_n, int symmetric) {
    TileAt r;
    r.b = t / per;
    const int k = (int)(t - r.b * per);
    if (symmetric) {
        int i = (int)((sqrtf(8.f * (float)k + 1.f) - 1.f) * 0.5f);
        while (i * (i + 1) / 2 > k) --i;
        while ((i + 1) * (i + 2) / 2 <= k) ++i;
        r.i = i;
        r.j = k - i * (i + 1) / 2;
    } else {
        r.i = k / tiles_n;
        r.j = k - r.i * tiles_n;
    }
    return r;
}

template <bool SPLIT>
__global__ void __launch_bounds__(kGemmThreads, 1)
    ortho_gemm_kernel(const __grid_constant__ OrthoGemm g, const __grid_constant__ GemmMaps maps,
                      const __grid_constant__ MuonTable tab, int per, int tiles_n, long long tiles) {
    constexpr int kStages = SPLIT ? kSplitStages : kHalfStages;
    constexpr int kPlanes = SPLIT ? 4 : 2; // P, Q or P hi, P lo, Q hi, Q lo
    constexpr int kStageBytes = kPlanes * kPlaneBytes;
    extern __shared__ char raw[];
    __shared__ GemmShared sh;
    const uint32_t stage0 = (smem_u32(raw) + 1023u) & ~1023u;
    const int warp = uniform_warp(), lane = threadIdx.x % 32;
    volatile int *abort = &sh.abort;

    if (warp == kEpilogueWarps && lane == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sh.full[s], 1);
            mbar_init(&sh.empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&sh.acc_full[a], 1);
            mbar_init(&sh.acc_empty[a], kEpilogueWarps);
        }
        sh.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kEpilogueWarps + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                     "r"(kTmemColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);

    const int kblocks = (g.K + kBK - 1) / kBK;
    const int total = kblocks * g.pairs;               // stages of a tile
    const int chunk = SPLIT ? kChunk : total;          // stages of an accumulation
    if (warp == kEpilogueWarps) {
        // the copies
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            long long loads = 0;
            bool ok = true;
            for (long long t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
                const TileAt at = tile_at(t, per, tiles_n, g.symmetric);
                if (tab.n > 0 && !muon_visible(tab, muon_tensor_of(tab, at.b), at.b)) continue;
                const int b = (int)at.b, i0 = at.i * kBM, j0 = at.j * kBN;
                for (int s = 0; s < total; ++s) {
                    const int pair = s >= kblocks, k0 = (s - pair * kblocks) * kBK;
                    ok = mbar_wait(&sh.empty[stage], phase ^ 1u, abort);
                    if (!ok) break;
                    const uint32_t dst = stage0 + stage * kStageBytes;
                    mbar_expect(&sh.full[stage], kStageBytes);
                    tma_load(dst, &maps.p_hi[pair], k0, i0, b, &sh.full[stage]);
                    if (SPLIT) tma_load(dst + kPlaneBytes, &maps.p_lo[pair], k0, i0, b, &sh.full[stage]);
#pragma unroll
                    for (int lo = 0; lo < (SPLIT ? 2 : 1); ++lo) {
                        const CUtensorMap *m = lo ? &maps.q_lo[pair] : &maps.q_hi[pair];
                        const uint32_t q = dst + (SPLIT ? 2 + lo : 1) * kPlaneBytes;
                        if (g.q_k_major) {
                            tma_load(q, m, k0, j0, b, &sh.full[stage]);
                        } else {
                            tma_load(q, m, j0, k0, b, &sh.full[stage]);
                            tma_load(q + kPlaneBytes / 2, m, j0 + 64, k0, b, &sh.full[stage]);
                        }
                    }
                    ++loads;
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (!ok) { // wait, with a limit, for the copies in flight
                const long long first = loads > kStages ? loads - kStages : 0;
                for (long long l = first; l < loads; ++l)
                    for (unsigned i = 0; i < kWaitLimit && !mbar_try(&sh.full[l % kStages], (uint32_t)(l / kStages) & 1u); ++i) {}
            }
        }
    } else if (warp == kEpilogueWarps + 1) {
        // the products
        const uint32_t leader = elect_leader();
        {
            const uint32_t idesc = mma_desc(kBN, g.q_k_major);
            const uint32_t q_step = g.q_k_major ? 32 / 16 : 2048 / 16; // 16 deep, in the descriptor's units
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            for (long long t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
                const TileAt at = tile_at(t, per, tiles_n, g.symmetric);
                if (tab.n > 0 && !muon_visible(tab, muon_tensor_of(tab, at.b), at.b)) continue;
                for (int s0 = 0; ok && s0 < total; s0 += chunk) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&sh.acc_empty[acc], acc_phase ^ 1u, abort));
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t d = tmem + acc * kBN;
                    const int s1 = min(total, s0 + chunk);
                    for (int s = s0; s < s1; ++s) {
                        ok = __all_sync(0xffffffffu, mbar_wait(&sh.full[stage], phase, abort));
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t src = stage0 + stage * kStageBytes;
                        const uint64_t p = operand_desc(src, true, 0);
                        const uint64_t q = operand_desc(src + (SPLIT ? 2 : 1) * kPlaneBytes, g.q_k_major, kPlaneBytes / 2);
                        const uint64_t lo = kPlaneBytes / 16; // from hi to lo
#pragma unroll
                        for (int k = 0; k < kBK / 16; ++k) {
                            mma_f16(d, p + k * 2, q + k * q_step, idesc, s > s0 || k > 0, leader);
                            if (SPLIT) {
                                mma_f16(d, p + k * 2, q + lo + k * q_step, idesc, true, leader);
                                mma_f16(d, p + lo + k * 2, q + k * q_step, idesc, true, leader);
                            }
                        }
                        mma_commit(&sh.empty[stage], leader);
                        if (++stage == kStages) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                    mma_commit(&sh.acc_full[acc], leader); // also after a wait that ran out: what was issued is waited for
                    acc ^= 1;
                    if (acc == 0) acc_phase ^= 1u;
                }
            }
        }
    } else {
        // the epilogue: warp w reads lanes 32 (w % 4) .., columns 64 (w / 4) ..
        const int row = 32 * (warp % 4) + lane, half = warp / 4;
        const bool poisoned = (g.epilogue == kEpiOut || g.epilogue == kEpiMuon) && *(volatile const int *)g.error != 0;
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        for (long long t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
            const TileAt at = tile_at(t, per, tiles_n, g.symmetric);
            const int tensor = tab.n > 0 ? muon_tensor_of(tab, at.b) : 0;
            if (tab.n > 0 && !muon_visible(tab, tensor, at.b)) continue;
            float v[64];
            for (int s0 = 0; s0 < total; s0 += chunk) {
                ok = __all_sync(0xffffffffu, mbar_wait(&sh.acc_full[acc], acc_phase, abort));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t src = tmem + ((uint32_t)(32 * (warp % 4)) << 16) + acc * kBN + half * 64;
                if (s0 == 0) {
                    tmem_load32(src, v);
                    tmem_load32(src + 32, v + 32);
                } else {
                    float u[32];
                    tmem_load32(src, u);
#pragma unroll
                    for (int c = 0; c < 32; ++c) v[c] += u[c];
                    tmem_load32(src + 32, u);
#pragma unroll
                    for (int c = 0; c < 32; ++c) v[32 + c] += u[c];
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.acc_empty[acc]);
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1u;
            }
            if (!ok) break;
            const int i = at.i * kBM + row, j = at.j * kBN + half * 64;
            if (i < g.M) {
                const bool mirror = g.symmetric && at.i != at.j;
                if (j < g.N) finish32(g, tab, tensor, at.b, i, j, mirror, poisoned, v);
                if (j + 32 < g.N) finish32(g, tab, tensor, at.b, i, j + 32, mirror, poisoned, v + 32);
            }
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == kEpilogueWarps + 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns) : "memory");
    if (threadIdx.x == 0 && sh.abort) atomicExch(g.error, 1);
}

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

template <bool SPLIT>
static int launch(const OrthoGemm &g, const GemmMaps &maps, const MuonTable &tab, cudaStream_t stream) {
    constexpr int smem = (SPLIT ? kSplitStages * 4 : kHalfStages * 2) * kPlaneBytes + 1024;
    const int tm = (g.M + kBM - 1) / kBM, tn = (g.N + kBN - 1) / kBN;
    const int per = g.symmetric ? tm * (tm + 1) / 2 : tm * tn;
    const long long tiles = g.batch * per;
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
        cudaFuncSetAttribute(ortho_gemm_kernel<SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
        return check_launch("ortho_gemm_kernel attributes");
    const unsigned blocks = (unsigned)(tiles < sms ? tiles : sms);
    ortho_gemm_kernel<SPLIT><<<blocks, kGemmThreads, smem, stream>>>(g, maps, tab, per, tn, tiles);
    return check_launch("ortho_gemm_kernel");
}

int ortho_gemm(const OrthoGemm &g, const MuonTable *table, cudaStream_t stream) {
    if (encode_fn() == nullptr) return set_error(kErrUnsupported, "orthogonalize: the driver offers no tensor maps");
    GemmMaps maps;
    for (int i = 0; i < g.pairs; ++i) {
        const int qr = g.q_k_major ? g.N : g.K, qc = g.q_k_major ? g.K : g.N, qb = g.q_k_major ? kBN : 64;
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
    return g.split ? launch<true>(g, maps, tab, stream) : launch<false>(g, maps, tab, stream);
}

} // namespace gsb
