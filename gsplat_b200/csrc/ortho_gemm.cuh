// Batched products of the Newton-Schulz iteration with their element-wise ends, on
// the fifth-generation tensor cores: one persistent block an SM, TMA into 128-byte-swizzled
// stages, tcgen05.mma into double-buffered TMEM accumulators, and eight warps that
// finish a tile while the next one is multiplied.
//
// A tile is 128 x BN of the result, 64 deep a stage. With SPLIT, a stage holds
// the hi and lo planes of both operands and feeds three products (hi hi, hi lo, lo hi);
// the sum is taken out of the tensor cores every kChunk stages and continued in
// registers, since their 32-bit adder truncates and the bias of a long sum of
// squares would be seen in the diagonal of A.
// A product of a middle-sized matrix takes about 8.5 us: 1.8 from the end of the launch before it, 2.2 until the first copies are
// there, 2 to 3 of products and 2 for the end ([257, 1000], 141 us in all).
// A launch follows the one before it without a gap: its blocks set up while that one ends (griddepcontrol).
#pragma once

#include <algorithm>
#include <cuda.h>

#include "ortho.cuh"
#include "tcgen05.cuh"

namespace gsb {

constexpr int kBM = 128, kBK = 64;
constexpr int kChunk = 4; // stages between two readings of the accumulator, split: a result 1.3e-6 off, 2.6e-6 with 8
                          // (FP32 GEMMs 2.5 to 4.8e-6)
// Products of hi alone deeper than kHiDepth (LONG) are read out every kHiChunk stages: the truncation takes 5e-8 of the sum at each
// of its additions (16 deep), 5e-5 in 16384, where the operands' 11 bits take 2e-4. Unread, the square of a row of 8 million
// was 0.7% short. The others are not read out, which is 1 to 2% faster.
constexpr int kHiDepth = 16384, kHiChunk = 32;
constexpr int kEpilogueWarps = 8;  // four lane quarters x two column halves
constexpr int kGemmThreads = 32 * (kEpilogueWarps + 2);
constexpr int kStagePitch = 33;    // floats a row of a warp's 32 x 32 values on their way out
constexpr int kOutStage = kEpilogueWarps * 32 * kStagePitch * 4;
constexpr int kMaxStages = 8;

// Bytes of a stage, and how many fit beside the epilogue's.
template <bool SPLIT, int BN> struct Stages {
    static constexpr int p = kBM * kBK * 2, q = BN * kBK * 2, bytes = (SPLIT ? 2 : 1) * (p + q);
    static constexpr int fit = (227 * 1024 - 1024 - 512 - kOutStage) / bytes;
    static constexpr int n = fit < kMaxStages ? fit : kMaxStages;
    static constexpr int smem = n * bytes + kOutStage + 1024;
};

struct GemmMaps {
    CUtensorMap p_hi[2], p_lo[2], q_hi[2], q_lo[2];
};

struct GemmShared {
    alignas(8) unsigned long long full[kMaxStages], empty[kMaxStages];
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

// Eight values of a row of planes, as they are stored.
struct Eight {
    uint4 hi, lo;
};
template <bool LO> __device__ __forceinline__ void unpack8(const Eight &r, float v[8]) {
    const __half2 *h = reinterpret_cast<const __half2 *>(&r.hi), *l = reinterpret_cast<const __half2 *>(&r.lo);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = __half22float2(h[i]);
        v[2 * i] = a.x;
        v[2 * i + 1] = a.y;
        if (LO) {
            const float2 b = __half22float2(l[i]);
            v[2 * i] += b.x;
            v[2 * i + 1] += b.y;
        }
    }
}
__device__ __forceinline__ Eight pack8(const float v[8]) {
    Eight r;
    __half2 *h = reinterpret_cast<__half2 *>(&r.hi), *l = reinterpret_cast<__half2 *>(&r.lo);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        const float2 f = __half22float2(h[i]);
        l[i] = __floats2half2_rn(v[2 * i] - f.x, v[2 * i + 1] - f.y);
    }
    return r;
}

// A warp's 32 x 32 values of planes, between a lane to a row (as the accumulator lies) and four
// lanes to a row's 64 bytes (as memory wants it: lane l has piece l % 4 of rows l / 4 + 8 k), through
// the warp's shared memory: hi, then lo, 2 KiB each, the pieces of a row permuted so that no banks meet.
__device__ __forceinline__ uint4 *stage_piece(float *stage, int plane, int row, int piece) {
    return reinterpret_cast<uint4 *>(stage) + plane * 128 + row * 4 + (piece ^ ((row >> 1) & 3));
}

struct TileAt {
    long long b;
    int i, j; // in tiles
};
// Tile t of the launch. Symmetric results list, by rows, the tiles with a column on or below the
// diagonal: of row block i the column tiles 0 .. i * kBM / BN (BN <= kBM: all of the diagonal block's).
template <int BN> __device__ __forceinline__ TileAt tile_at(long long t, int per, int tiles_n, int symmetric) {
    constexpr int w = kBM / BN; // column tiles of a row block
    TileAt r;
    r.b = t / per;
    const int k = (int)(t - r.b * per);
    if (symmetric) { // rows 0 .. i - 1 hold w i (i + 1) / 2 tiles
        int i = (int)((sqrtf(8.f * (float)(k / w) + 1.f) - 1.f) * 0.5f);
        while (w * i * (i + 1) / 2 > k) --i;
        while (w * (i + 1) * (i + 2) / 2 <= k) ++i;
        r.i = i;
        r.j = k - w * i * (i + 1) / 2;
    } else {
        r.i = k / tiles_n;
        r.j = k - r.i * tiles_n;
    }
    return r;
}

// What an epilogue reads and writes.
template <bool SPLIT, int EPI> struct Epilogue {
    static constexpr bool symmetric = EPI == kEpiGram || EPI == kEpiSquare || EPI == kEpiSym || EPI == kEpiAnti;
    static constexpr bool element = EPI != kEpiGram && EPI != kEpiSym; // reads e
    static constexpr bool row_diag = element;                         // and the diagonal at its row
    static constexpr bool col_diag = EPI == kEpiSquare || EPI == kEpiAnti;
    static constexpr bool element_lo = SPLIT || !symmetric;
    static constexpr bool to_planes = EPI != kEpiOut && EPI != kEpiMuon;
    static constexpr bool out_lo = SPLIT || EPI == kEpiApply;
};

// Where the last step's 32 x 32 values go: a lane's n values, `step` apart. Neighbouring lanes are at
// neighbouring places of the tensor: with a transposed tensor the lanes' rows are, and a lane has its row's values;
// else a lane has a column, and the values are turned through shared memory.
struct OutAt {
    void *p;
    size_t at, step;
    int n, dtype;
    bool turned;
};
template <int EPI>
__device__ __forceinline__ OutAt out_at(const OrthoGemm &g, const MuonTable &tab, int tensor, long long b, int i, int j, int lane) {
    OutAt r;
    r.turned = EPI == kEpiMuon ? tab.transposed[tensor] : (bool)g.transposed;
    r.p = EPI == kEpiMuon ? tab.param[tensor] : g.y;
    r.dtype = EPI == kEpiMuon ? tab.dtype : g.dtype;
    r.at = (size_t)(b - (EPI == kEpiMuon ? tab.first[tensor] : 0)) * g.M * g.N +
           (r.turned ? (size_t)j * g.M + i : (size_t)(i - lane) * g.N + j + lane);
    r.step = r.turned ? g.M : g.N;
    r.n = r.turned ? (i < g.M ? g.N - j : 0) : (lane < g.N - j ? g.M - (i - lane) : 0);
    return r;
}
// The parameters there, as they are stored (a 16-bit type in the low half), read together before they are needed: a
// conversion beside each would wait for it.
template <int EPI>
__device__ __forceinline__ void fetch_params(const OrthoGemm &g, const MuonTable &tab, int tensor, long long b, int i, int j, int lane,
                                             uint32_t p[32]) {
    if (EPI != kEpiMuon) return;
    const OutAt from = out_at<EPI>(g, tab, tensor, b, i, j, lane);
    if (from.dtype == kOrthoF32) {
        const uint32_t *at = static_cast<const uint32_t *>(from.p) + from.at;
#pragma unroll
        for (int k = 0; k < 32; ++k) p[k] = k < from.n ? at[k * from.step] : 0u;
    } else {
        const unsigned short *at = static_cast<const unsigned short *>(from.p) + from.at;
#pragma unroll
        for (int k = 0; k < 32; ++k) p[k] = k < from.n ? at[k * from.step] : 0u;
    }
}
template <typename T> __device__ __forceinline__ float stored_as(uint32_t v);
template <> __device__ __forceinline__ float stored_as<float>(uint32_t v) { return __uint_as_float(v); }
template <> __device__ __forceinline__ float stored_as<__nv_bfloat16>(uint32_t v) { return __uint_as_float(v << 16); }
template <> __device__ __forceinline__ float stored_as<__half>(uint32_t v) { return __half2float(__ushort_as_half((unsigned short)v)); }

template <typename T, bool MUON>
__device__ __forceinline__ void put_out(const OutAt &to, const float v[32], const uint32_t p[32], const float *stage, int lane, float lr,
                                        float decay, bool poisoned) {
    T *at = static_cast<T *>(to.p) + to.at;
#pragma unroll
    for (int k = 0; k < 32; ++k) {
        if (k >= to.n) continue;
        float r = to.turned ? v[k] : stage[k * kStagePitch + lane];
        if (poisoned) r = NAN;
        at[k * to.step] = from_f32<T>(MUON ? muon_param(stored_as<T>(p[k]), r, lr, decay) : r);
    }
}

// The epilogue of 32 columns from j of a lane's row i, the accumulator's values in v. di, dj: the diagonal
// at the row, and at the lane's one of the columns. stage: the warp's shared memory, with the element-wise operand.
template <bool SPLIT, int EPI>
__device__ __forceinline__ void finish32(const OrthoGemm &g, const MuonTable &tab, int tensor, long long b, int i, int j, int lane,
                                         float v[32], const uint32_t p[32], float di, float dj, bool mirror, bool poisoned, float *stage) {
    using E = Epilogue<SPLIT, EPI>;
    const bool in_rows = i < g.M;
#pragma unroll
    for (int c = 0; c < 32; c += 8) {
        float *w = v + c, x[8];
        if (E::element) {
            Eight r;
            r.hi = *stage_piece(stage, 0, lane, c / 8);
            if (E::element_lo) r.lo = *stage_piece(stage, 1, lane, c / 8);
            unpack8<E::element_lo>(r, x);
        }
        float on = 0.f;
        bool diagonal = false;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const bool here = (EPI == kEpiGram || EPI == kEpiSquare) && i == j + c + k;
            on = here ? w[k] : on;
            diagonal |= here;
            if (EPI == kEpiGram || EPI == kEpiSym) {
                w[k] *= g.c[0];
            } else if (E::col_diag) {
                const float d = __shfl_sync(0xffffffffu, dj, c + k);
                w[k] = fmaf(fmaf(g.c[1], di + d, g.c[0]), x[k], g.c[2] * w[k]);
            } else {
                w[k] = fmaf(g.c[0] + di, x[k], g.c[1] * w[k]) * g.c[2];
            }
            if (here) w[k] = 0.f;
        }
        if (diagonal && in_rows)
            g.diag_out[(size_t)b * g.M + i] = EPI == kEpiGram ? g.c[1] * on : fmaf(g.c[3], di, fmaf(g.c[4] * di, di, g.c[5] * on));
        if (E::to_planes) { // in the place of the lane's own piece of e
            const Eight r = pack8(w);
            *stage_piece(stage, 0, lane, c / 8) = r.hi;
            if (E::out_lo) *stage_piece(stage, 1, lane, c / 8) = r.lo;
            if (E::symmetric && mirror && in_rows && j + c < g.N) { // blocks off the diagonal have all their columns
                __half *mh = g.out.hi + (size_t)b * g.out.stride + (size_t)(j + c) * g.out.ld + i;
                __half *ml = g.out.lo + (mh - g.out.hi);
                const __half *h = reinterpret_cast<const __half *>(&r.hi), *l = reinterpret_cast<const __half *>(&r.lo);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    mh[(size_t)k * g.out.ld] = h[k];
                    if (E::out_lo) ml[(size_t)k * g.out.ld] = l[k];
                }
            }
        }
    }
    if (E::to_planes) {
        __syncwarp();
        const int first = i - lane + lane / 4, col = j + 8 * (lane % 4);
        const size_t at = (size_t)b * g.out.stride + (size_t)first * g.out.ld + col;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (first + 8 * k < g.M && col < g.N) {
                *reinterpret_cast<uint4 *>(g.out.hi + at + (size_t)(8 * k) * g.out.ld) = *stage_piece(stage, 0, lane / 4 + 8 * k, lane % 4);
                if (E::out_lo)
                    *reinterpret_cast<uint4 *>(g.out.lo + at + (size_t)(8 * k) * g.out.ld) = *stage_piece(stage, 1, lane / 4 + 8 * k, lane % 4);
            }
        }
        __syncwarp();
    }
    if (E::to_planes) return;
    const OutAt to = out_at<EPI>(g, tab, tensor, b, i, j, lane);
    const float lr = EPI == kEpiMuon ? tab.lr[tensor] : 0.f, decay = EPI == kEpiMuon ? tab.decay[tensor] : 0.f;
    if (!to.turned) {
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 32; ++k) stage[lane * kStagePitch + k] = v[k];
        __syncwarp();
    }
    if (to.dtype == kOrthoF32) put_out<float, EPI == kEpiMuon>(to, v, p, stage, lane, lr, decay, poisoned);
    else if (to.dtype == kOrthoBF16) put_out<__nv_bfloat16, EPI == kEpiMuon>(to, v, p, stage, lane, lr, decay, poisoned);
    else put_out<__half, EPI == kEpiMuon>(to, v, p, stage, lane, lr, decay, poisoned);
}

// A wait of the last product ran out in this block: its epilogue warps write NaN to its 128 rows, from row0, of each of its
// tiles, of which one may have been finished from a sum that was not whole.
template <int EPI, int BN, int ROWS>
__device__ void give_up(const OrthoGemm &g, const MuonTable &tab, long long t, long long tiles, long long stride, int per, int tiles_n,
                        int row0) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, row = row0 + 32 * (warp % 4) + lane, col = warp / 4 * (BN / 2);
    for (; t < tiles; t += stride) {
        const TileAt at = tile_at<kBM>(t, per, tiles_n, false);
        const int tensor = tab.n > 0 ? muon_tensor_of(tab, at.b) : 0;
        if (tab.n > 0 && !muon_visible(tab, tensor, at.b)) continue;
#pragma unroll 1
        for (int c = 0; c < BN / 2; c += 32) {
            const OutAt to = out_at<EPI>(g, tab, tensor, at.b, at.i * ROWS + row, at.j * BN + col + c, lane);
#pragma unroll 1
            for (int k = 0; k < to.n && k < 32; ++k) {
                const size_t e = to.at + k * to.step;
                if (to.dtype == kOrthoF32) static_cast<float *>(to.p)[e] = NAN;
                else if (to.dtype == kOrthoBF16) static_cast<__nv_bfloat16 *>(to.p)[e] = from_f32<__nv_bfloat16>(NAN);
                else static_cast<__half *>(to.p)[e] = from_f32<__half>(NAN);
            }
        }
    }
}

// The operand e of the warp's 32 rows and 32 columns from j, four lanes to a row; nothing past the matrix.
template <bool SPLIT, int EPI>
__device__ __forceinline__ void fetch32(const OrthoGemm &g, long long b, int row0, int j, int lane, Eight e[4]) {
    using E = Epilogue<SPLIT, EPI>;
    if (!E::element) return;
    const int first = row0 + lane / 4, col = j + 8 * (lane % 4);
    const size_t at = (size_t)b * g.e.stride + (size_t)first * g.e.ld + col;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (first + 8 * k < g.M && col < g.N) {
            e[k].hi = *reinterpret_cast<const uint4 *>(g.e.hi + at + (size_t)(8 * k) * g.e.ld);
            if (E::element_lo) e[k].lo = *reinterpret_cast<const uint4 *>(g.e.lo + at + (size_t)(8 * k) * g.e.ld);
        }
    }
}

// And from the registers to the warp's shared memory, for finish32.
template <bool SPLIT, int EPI> __device__ __forceinline__ void stage32(float *stage, int lane, const Eight e[4]) {
    using E = Epilogue<SPLIT, EPI>;
    __syncwarp();
    if (!E::element) return;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        *stage_piece(stage, 0, lane / 4 + 8 * k, lane % 4) = e[k].hi;
        if (E::element_lo) *stage_piece(stage, 1, lane / 4 + 8 * k, lane % 4) = e[k].lo;
    }
    __syncwarp();
}

__device__ __forceinline__ uint32_t block_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
}
// The leader's (rank 0's) copy of an address of this block's shared memory, and a store to it.
__device__ __forceinline__ uint32_t at_leader(uint32_t addr) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void store_at(uint32_t addr, float4 v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

// DEEP: the blocks of a cluster share a tile, each with a part of the depth. All but the leader leave their
// sums in its shared memory (where its stages were), and it adds them in the order of the blocks and finishes
// the tile; a launch then has one tile a cluster. For long contractions with few tiles (A of a
// short matrix), whose blocks would otherwise work through the depth alone.
template <bool SPLIT, int BN, int EPI, bool DEEP, bool LONG>
__global__ void __launch_bounds__(kGemmThreads, 1)
    ortho_gemm_kernel(const __grid_constant__ OrthoGemm g, const __grid_constant__ GemmMaps maps,
                      const __grid_constant__ MuonTable tab, int per, int tiles_n, long long tiles) {
    using Stage = Stages<SPLIT, BN>;
    constexpr int kStages = Stage::n;
    using E = Epilogue<SPLIT, EPI>;
    constexpr bool kSymmetric = E::symmetric, kQDepthMajor = kSymmetric;
    constexpr int W = BN / 2; // columns of a warp
    extern __shared__ char raw[];
    __shared__ GemmShared sh;
    const uint32_t stage0 = (smem_u32(raw) + 1023u) & ~1023u;
    const int warp = uniform_warp(), lane = threadIdx.x % 32;
    volatile int *abort = &sh.abort;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); // the next product's blocks may set up; they wait below
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
    if (warp == kEpilogueWarps && lane < 8) { // the tensor maps: fetched while the launch before this one ends
        const CUtensorMap *m = &maps.p_hi[0] + lane;
        asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
    }
    if (warp == kEpilogueWarps + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                     "r"(2 * BN)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
    asm volatile("griddepcontrol.wait;" ::: "memory"); // for what the launches before this one wrote

    const int kblocks = (g.K + kBK - 1) / kBK;
    const int ranks = DEEP ? (int)cluster_size() : 1, rank = DEEP ? (int)block_rank() : 0;
    const int all = kblocks * g.pairs;                                              // stages of a tile
    const int begin = DEEP ? all * rank / ranks : 0, end = DEEP ? all * (rank + 1) / ranks : all; // this block's
    const int chunk = SPLIT ? kChunk : LONG ? kHiChunk : end - begin;                                // stages of an accumulation
    const long long first = DEEP ? blockIdx.x / ranks : blockIdx.x, stride = DEEP ? gridDim.x / ranks : gridDim.x;
    // whether the cluster's one tile is worked on, by all of its blocks' warps
    const bool shared_tile = DEEP && !(tab.n > 0 && !muon_visible(tab, muon_tensor_of(tab, first / per), first / per));
    if (warp == kEpilogueWarps) {
        // the copies
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            long long loads = 0;
            bool ok = true;
            for (long long t = first; ok && t < tiles; t += stride) {
                const TileAt at = tile_at<BN>(t, per, tiles_n, kSymmetric);
                if (tab.n > 0 && !muon_visible(tab, muon_tensor_of(tab, at.b), at.b)) continue;
                const int b = (int)at.b, i0 = at.i * kBM, j0 = at.j * BN;
                for (int s = begin; s < end; ++s) {
                    const int pair = s >= kblocks, k0 = (s - pair * kblocks) * kBK;
                    ok = mbar_wait(&sh.empty[stage], phase ^ 1u, abort);
                    if (!ok) break;
                    uint32_t dst = stage0 + stage * Stage::bytes;
                    unsigned long long *bar = &sh.full[stage];
                    mbar_expect(bar, Stage::bytes);
                    tma_load(dst, &maps.p_hi[pair], k0, i0, b, bar);
                    if (SPLIT) tma_load(dst + Stage::p, &maps.p_lo[pair], k0, i0, b, bar);
                    dst += (SPLIT ? 2 : 1) * Stage::p;
#pragma unroll
                    for (int lo = 0; lo < (SPLIT ? 2 : 1); ++lo) {
                        const CUtensorMap *m = lo ? &maps.q_lo[pair] : &maps.q_hi[pair];
                        if (kQDepthMajor) {
                            tma_load(dst + lo * Stage::q, m, k0, j0, b, bar);
                        } else {
#pragma unroll
                            for (int c = 0; c < BN / 64; ++c) tma_load(dst + lo * Stage::q + c * kBK * 128, m, j0 + 64 * c, k0, b, bar);
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
        if (DEEP && shared_tile) {
            __syncwarp();
            cluster_barrier();
            cluster_barrier();
        }
    } else if (warp == kEpilogueWarps + 1) {
        // the products
        const uint32_t leader = elect_leader();
        constexpr uint32_t q_step = kQDepthMajor ? 32 / 16 : 2048 / 16; // 16 deep, in the descriptor's units
        const uint32_t idesc = mma_desc(BN, kQDepthMajor);
        int stage = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true, issued = false;
        for (long long t = first; ok && t < tiles; t += stride) {
            const TileAt at = tile_at<BN>(t, per, tiles_n, kSymmetric);
            if (tab.n > 0 && !muon_visible(tab, muon_tensor_of(tab, at.b), at.b)) continue;
            for (int s0 = begin; ok && s0 < end; s0 += chunk) {
                ok = __all_sync(0xffffffffu, mbar_wait(&sh.acc_empty[acc], acc_phase ^ 1u, abort));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t d = tmem + acc * BN;
                const int s1 = min(end, s0 + chunk);
                for (int s = s0; s < s1; ++s) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&sh.full[stage], phase, abort));
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t src = stage0 + stage * Stage::bytes;
                    const uint64_t p = operand_desc(src, true, 0);
                    const uint64_t q = operand_desc(src + (SPLIT ? 2 : 1) * Stage::p, kQDepthMajor, kBK * 128);
                    constexpr uint64_t p_lo = Stage::p / 16, q_lo = Stage::q / 16; // from hi to lo
#pragma unroll
                    for (int k = 0; k < kBK / 16; ++k) {
                        mma_f16(d, p + k * 2, q + k * q_step, idesc, s > s0 || k > 0, leader);
                        if (SPLIT) {
                            mma_f16(d, p + k * 2, q + q_lo + k * q_step, idesc, true, leader);
                            mma_f16(d, p + p_lo + k * 2, q + k * q_step, idesc, true, leader);
                        }
                    }
                    mma_commit(&sh.empty[stage], leader);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) __threadfence_block(); // the epilogue finds the abort word set behind this barrier
                mma_commit(&sh.acc_full[acc], leader);
                issued = true;
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1u;
            }
        }
        if (!ok && issued) { // wait, with a limit, for the products in flight, which come to an end in their order
            const uint32_t last_phase = acc == 0 ? acc_phase ^ 1u : acc_phase;
            for (unsigned i = 0; i < kWaitLimit && !mbar_try(&sh.acc_full[acc ^ 1], last_phase); ++i) {}
        }
        if (DEEP && shared_tile) {
            __syncwarp();
            cluster_barrier();
            cluster_barrier();
        }
    } else {
        // the epilogue: warp w has rows 32 (w % 4) .., columns W (w / 4) ..
        const int row = 32 * (warp % 4) + lane, half = warp / 4;
        float *out_stage = reinterpret_cast<float *>(raw + (stage0 - smem_u32(raw)) + kStages * Stage::bytes) + warp * 32 * kStagePitch;
        const bool poisoned = !E::to_planes && *(volatile const int *)g.error != 0;
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        for (long long t = first; ok && t < tiles; t += stride) {
            const TileAt at = tile_at<BN>(t, per, tiles_n, kSymmetric);
            const int tensor = tab.n > 0 ? muon_tensor_of(tab, at.b) : 0;
            if (tab.n > 0 && !muon_visible(tab, tensor, at.b)) continue;
            const int i = at.i * kBM + row, j = at.j * BN + half * W;
            // what the epilogue needs is read while the products run
            Eight e[4];
            float di = 0.f, dj[W / 32] = {};
            if (E::row_diag && i < g.M) di = g.diag_in[(size_t)at.b * g.M + i];
#pragma unroll
            for (int c = 0; c < W / 32; ++c) {
                if (E::col_diag && j + 32 * c + lane < g.N) dj[c] = g.diag_in[(size_t)at.b * g.M + j + 32 * c + lane];
            }
            fetch32<SPLIT, EPI>(g, at.b, i - lane, j, lane, e);
            float v[W];
            for (int s0 = begin; s0 < end; s0 += chunk) {
                ok = __all_sync(0xffffffffu, mbar_wait(&sh.acc_full[acc], acc_phase, abort));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t src = tmem + ((uint32_t)(32 * (warp % 4)) << 16) + acc * BN + half * W;
#pragma unroll
                for (int c = 0; c < W; c += 32) {
                    float u[32];
                    tmem_load32(src + c, u);
#pragma unroll
                    for (int k = 0; k < 32; ++k) v[c + k] = s0 == begin ? u[k] : v[c + k] + u[k];
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.acc_empty[acc]);
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1u;
            }
            if (DEEP) { // rank r's sums at r - 1 of [ranks - 1][warp][W / 4][lane], four columns each
                const uint32_t sums = stage0 + (uint32_t)(warp * (W / 4) * 32 + lane) * 16;
                constexpr uint32_t block = kEpilogueWarps * (W / 4) * 32 * 16;
                __syncwarp();
                cluster_barrier(); // the leader's stages are done with
                if (rank > 0) {
                    const uint32_t to = at_leader(sums) + (rank - 1) * block;
#pragma unroll
                    for (int c = 0; c < W; c += 4) store_at(to + c / 4 * 512, make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]));
                }
                cluster_barrier();
                if (rank > 0) break;
                for (int r = 1; r < ranks; ++r) {
#pragma unroll
                    for (int c = 0; c < W; c += 4) {
                        float4 f;
                        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w)
                                     : "r"(sums + (r - 1) * block + c / 4 * 512)
                                     : "memory");
                        v[c] += f.x, v[c + 1] += f.y, v[c + 2] += f.z, v[c + 3] += f.w;
                    }
                }
            }
            if (!ok) break;
            const bool mirror = (at.j * BN) / kBM != at.i; // off the diagonal block
#pragma unroll
            for (int c = 0; c < W / 32; ++c) {
                uint32_t p[32];
                fetch_params<EPI>(g, tab, tensor, at.b, i, j + 32 * c, lane, p);
                stage32<SPLIT, EPI>(out_stage, lane, e);
                if (c + 1 < W / 32) fetch32<SPLIT, EPI>(g, at.b, i - lane, j + 32 * (c + 1), lane, e);
                finish32<SPLIT, EPI>(g, tab, tensor, at.b, i, j + 32 * c, lane, v + 32 * c, p, di, dj[c], mirror, poisoned, out_stage);
            }
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (!E::to_planes && warp < kEpilogueWarps && *abort) give_up<EPI, BN, kBM>(g, tab, blockIdx.x, tiles, gridDim.x, per, tiles_n, 0);
    if (warp == kEpilogueWarps + 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN) : "memory");
    if (threadIdx.x == 0 && sh.abort) atomicExch(g.error, 1);
}

// Blocks that share a tile's depth: as many as there are SMs for, as fit their sums beside each other in the
// leader's stages, and as have 2 us of products each (4 or 12 stages), which is what meeting costs. With
// more tiles than the GPU has groups of SMs that a cluster must fit in (8), a power of two, and fours on 7/8 of the
// SMs: the groups' sizes leave some of them without work.
template <bool SPLIT, int BN> static int tile_ranks(const OrthoGemm &g, long long tiles, int sms) {
    if (g.epilogue != kEpiGram && g.epilogue != kEpiSym) return 1;
    constexpr int most = Stages<SPLIT, BN>::n * Stages<SPLIT, BN>::bytes / (kBM * BN * 4) + 1;
    const int stages = (g.K + kBK - 1) / kBK * g.pairs;
    const int ranks = (int)std::min<long long>({sms / tiles, stages / (SPLIT ? 4 : 12), most, 8});
    return ranks < 2 ? 1 : tiles <= 8 ? ranks : ranks >= 4 && 4 * tiles <= sms * 7 / 8 ? 4 : 2;
}

template <bool SPLIT, int BN, int EPI, bool LONG>
static int launch_depth(const OrthoGemm &g, const GemmMaps &maps, const MuonTable &tab, int per, int tn, long long tiles,
                      int sms, cudaStream_t stream) {
    constexpr int smem = Stages<SPLIT, BN>::smem;
    const int ranks = tile_ranks<SPLIT, BN>(g, tiles, sms);
    constexpr bool kDeep = EPI == kEpiGram || EPI == kEpiSym;
    if constexpr (kDeep) {
        if (ranks > 1) {
            auto *kernel = ortho_gemm_kernel<SPLIT, BN, EPI, true, LONG>;
            if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
                return check_launch("ortho_gemm_kernel attributes");
            return launch_clusters_after(kernel, ranks, (unsigned)(tiles * ranks), kGemmThreads, smem, stream, "ortho_gemm_kernel", g, maps,
                                         tab, per, tn, tiles);
        }
    }
    auto *kernel = ortho_gemm_kernel<SPLIT, BN, EPI, false, LONG>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
        return check_launch("ortho_gemm_kernel attributes");
    return launch_after(kernel, (unsigned)(tiles < sms ? tiles : sms), kGemmThreads, smem, stream, "ortho_gemm_kernel", g, maps, tab,
                        per, tn, tiles);
}

template <bool SPLIT, int BN, int EPI>
static int launch_one(const OrthoGemm &g, const GemmMaps &maps, const MuonTable &tab, int per, int tn, long long tiles,
                      int sms, cudaStream_t stream) {
    // (B and X are as wide as they are deep, at least, and then never take 64 columns)
    constexpr bool kLong = !SPLIT && (BN == 128 || EPI == kEpiGram);
    if (kLong && g.K > kHiDepth) return launch_depth<SPLIT, BN, EPI, kLong>(g, maps, tab, per, tn, tiles, sms, stream);
    return launch_depth<SPLIT, BN, EPI, false>(g, maps, tab, per, tn, tiles, sms, stream);
}

template <bool SPLIT, int BN>
int ortho_gemm_launch(const OrthoGemm &g, const GemmMaps &maps, const MuonTable &tab, int sms, cudaStream_t stream) {
    const int tm = (g.M + kBM - 1) / kBM, tn = (g.N + BN - 1) / BN;
    int per = tm * tn;
    if (g.symmetric) { // less the last row block's tiles past the last column
        constexpr int w = kBM / BN;
        per = w * tm * (tm + 1) / 2 - (w * tm - tn);
    }
    const long long tiles = g.batch * per;
    switch (g.epilogue) {
    case kEpiGram: return launch_one<SPLIT, BN, kEpiGram>(g, maps, tab, per, tn, tiles, sms, stream);
    case kEpiSquare: return launch_one<SPLIT, BN, kEpiSquare>(g, maps, tab, per, tn, tiles, sms, stream);
    case kEpiApply: return launch_one<SPLIT, BN, kEpiApply>(g, maps, tab, per, tn, tiles, sms, stream);
    case kEpiOut: return launch_one<SPLIT, BN, kEpiOut>(g, maps, tab, per, tn, tiles, sms, stream);
    case kEpiMuon: return launch_one<SPLIT, BN, kEpiMuon>(g, maps, tab, per, tn, tiles, sms, stream);
    default: break;
    }
    if constexpr (SPLIT) {
        if (g.epilogue == kEpiSym) return launch_one<SPLIT, BN, kEpiSym>(g, maps, tab, per, tn, tiles, sms, stream);
        return launch_one<SPLIT, BN, kEpiAnti>(g, maps, tab, per, tn, tiles, sms, stream);
    }
    return set_error(kErrUnsupported, "orthogonalize: a backward product of hi planes alone");
}

extern template int ortho_gemm_launch<true, 128>(const OrthoGemm &, const GemmMaps &, const MuonTable &, int, cudaStream_t);
extern template int ortho_gemm_launch<false, 128>(const OrthoGemm &, const GemmMaps &, const MuonTable &, int, cudaStream_t);
extern template int ortho_gemm_launch<true, 64>(const OrthoGemm &, const GemmMaps &, const MuonTable &, int, cudaStream_t);
extern template int ortho_gemm_launch<false, 64>(const OrthoGemm &, const GemmMaps &, const MuonTable &, int, cudaStream_t);

} // namespace gsb
