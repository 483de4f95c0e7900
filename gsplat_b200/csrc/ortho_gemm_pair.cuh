// The tiled products for large matrices: a pair of SMs multiplies a 256 x 256 tile together
// (tcgen05 cta_group::2). Each holds 128 rows of P and 128 of Q's 256 columns, and reads half as many operand
// bytes from its shared memory for a product as with a tile of its own: a 128 x 128 tile
// wants 126 bytes a cycle for its operands and 85 to 123 for the copies that fill its stages, of an SM's 128.
// Measured at 4096 x 4096: A 150 us, B 170, X 305 split (72% of cycles with the tensor cores at work; three products each),
// and 68 for X of 2048 x 8192 with hi alone, where the L2's bytes bound it.
// The rest is as in ortho_gemm.cuh: the leader (rank 0) issues the products for both; the copies of both are
// counted on the leader's barriers, and its commits free the stages and hand over the accumulators of both.
#pragma once

#include <atomic>

#include "ortho_gemm.cuh"

namespace gsb {

constexpr int kPair = 256;   // rows and columns of a tile
// Stages between two readings of the accumulator, split (4 cost 8% of a product). Of hi alone sums are not read out, so that they
// need no registers and a warp finishes 32 columns at a time (with registers for the sum [2048, 8192] took 1047 us instead of
// 752); those deeper than kHiDepth are left to the tiles of one SM.
constexpr int kPairChunk = 8;
// Split sums go on in 128 registers of an epilogue thread, more than three warpgroups at 168 leave it: the
// warpgroup of the copies and products gives 112 of its own. 2 x 224 + 56 = 3 x 168.
constexpr int kPairThreads = 384, kPairRegisters = 168, kEpilogueRegisters = 224, kIssueRegisters = 56;

constexpr int kPairUnfit = 1; // of a launch: the kernel was built with other registers. Tiles of one SM serve

template <bool SPLIT> struct PairStages {
    static constexpr int plane = 128 * kBK * 2, bytes = (SPLIT ? 4 : 2) * plane;
    static constexpr int n = (227 * 1024 - 1024 - 512 - kOutStage) / bytes;
    static constexpr int smem = n * bytes + kOutStage + 1024;
};

__device__ __forceinline__ void arrive_at(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// A copy into this block's shared memory, counted on the leader's barrier.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate, uint32_t leader) {
    asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %4, 0;\n setp.ne.u32 q, %5, 0;\n"
                 " @q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(leader)
                 : "memory");
}
// Arrives at this barrier of both blocks when the products so far are done.
__device__ __forceinline__ void commit_pair(unsigned long long *bar, uint32_t leader) {
    asm volatile("{\n .reg .pred q;\n setp.ne.u32 q, %2, 0;\n"
                 " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}" ::"r"(smem_u32(bar)),
                 "h"((uint16_t)3), "r"(leader)
                 : "memory");
}

// A wait of this block ran out: the other block's abort word is set too, before what this warp does next can be seen there.
// Both blocks stay until the last barrier.
__device__ __forceinline__ void abort_other(volatile int *abort, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(const_cast<int *>(abort))), "r"(rank ^ 1u));
    asm volatile("st.shared::cluster.u32 [%0], %1;\n fence.acq_rel.cluster;" ::"r"(at), "r"(1u) : "memory");
}

template <bool SPLIT, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    ortho_pair_kernel(const __grid_constant__ OrthoGemm g, const __grid_constant__ GemmMaps maps,
                      const __grid_constant__ MuonTable tab, int per, int tiles_n, long long tiles) {
    using Stage = PairStages<SPLIT>;
    using E = Epilogue<SPLIT, EPI>;
    constexpr int kStages = Stage::n;
    constexpr bool kSymmetric = E::symmetric, kQDepthMajor = kSymmetric;
    constexpr int W = kPair / 2; // columns of a warp
    extern __shared__ char raw[];
    __shared__ GemmShared sh;
    const uint32_t stage0 = (smem_u32(raw) + 1023u) & ~1023u;
    const int warp = uniform_warp(), lane = threadIdx.x % 32;
    const uint32_t rank = block_rank();
    const long long first = blockIdx.x / 2, pairs = gridDim.x / 2;
    volatile int *abort = &sh.abort;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (warp == kEpilogueWarps && lane == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sh.full[s], 1);
            mbar_init(&sh.empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&sh.acc_full[a], 1);
            mbar_init(&sh.acc_empty[a], 2 * kEpilogueWarps);
        }
        sh.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kEpilogueWarps && lane < 8) {
        const CUtensorMap *m = &maps.p_hi[0] + lane;
        asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
    }
    if (warp == kEpilogueWarps + 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(2 * kPair) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_barrier();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const int kblocks = (g.K + kBK - 1) / kBK;
    const int total = kblocks * g.pairs;
    const int chunk = SPLIT ? kPairChunk : total;
    if (warp >= kEpilogueWarps) {
    if (SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegisters));
    if (warp == kEpilogueWarps) {
        // the copies of this block
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (long long t = first; ok && t < tiles; t += pairs) {
                const TileAt at = tile_at<kBM>(t, per, tiles_n, kSymmetric);
                if (tab.n > 0 && !muon_visible(tab, muon_tensor_of(tab, at.b), at.b)) continue;
                const int b = (int)at.b, i0 = at.i * kPair + (int)rank * 128, j0 = at.j * kPair + (int)rank * 128;
                for (int s = 0; s < total; ++s) {
                    const int pair = s >= kblocks, k0 = (s - pair * kblocks) * kBK;
                    ok = mbar_wait(&sh.empty[stage], phase ^ 1u, abort);
                    if (!ok) break;
                    uint32_t dst = stage0 + stage * Stage::bytes;
                    const uint32_t bar = at_leader(smem_u32(&sh.full[stage]));
                    if (rank == 0) mbar_expect(&sh.full[stage], 2 * Stage::bytes);
                    tma_load_pair(dst, &maps.p_hi[pair], k0, i0, b, bar);
                    if (SPLIT) tma_load_pair(dst + Stage::plane, &maps.p_lo[pair], k0, i0, b, bar);
                    dst += (SPLIT ? 2 : 1) * Stage::plane;
#pragma unroll
                    for (int lo = 0; lo < (SPLIT ? 2 : 1); ++lo) {
                        const CUtensorMap *m = lo ? &maps.q_lo[pair] : &maps.q_hi[pair];
                        if (kQDepthMajor) {
                            tma_load_pair(dst + lo * Stage::plane, m, k0, j0, b, bar);
                        } else {
                            tma_load_pair(dst + lo * Stage::plane, m, j0, k0, b, bar);
                            tma_load_pair(dst + lo * Stage::plane + kBK * 128, m, j0 + 64, k0, b, bar);
                        }
                    }
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (!ok) abort_other(abort, rank);
            // a wait ran out: the copies in flight, counted on the leader's barriers, land within this time
            for (int i = 0; !ok && i < 10000; ++i) __nanosleep(1000);
        }
    } else if (warp == kEpilogueWarps + 1) {
        // the products of both, by the leader
        if (rank == 0) {
            const uint32_t leader = elect_leader();
            constexpr uint32_t q_step = kQDepthMajor ? 32 / 16 : 2048 / 16;
            constexpr uint32_t idesc = 1u << 4 | (kQDepthMajor ? 0u : 1u << 16) | (uint32_t)(kPair / 8) << 17 | (uint32_t)(kPair / 16) << 24;
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true, issued = false;
            for (long long t = first; ok && t < tiles; t += pairs) {
                const TileAt at = tile_at<kBM>(t, per, tiles_n, kSymmetric);
                if (tab.n > 0 && !muon_visible(tab, muon_tensor_of(tab, at.b), at.b)) continue;
                for (int s0 = 0; ok && s0 < total; s0 += chunk) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&sh.acc_empty[acc], acc_phase ^ 1u, abort));
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t d = tmem + acc * kPair;
                    const int s1 = min(total, s0 + chunk);
                    for (int s = s0; s < s1; ++s) {
                        ok = __all_sync(0xffffffffu, mbar_wait(&sh.full[stage], phase, abort));
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t src = stage0 + stage * Stage::bytes;
                        const uint64_t p = operand_desc(src, true, 0);
                        const uint64_t q = operand_desc(src + (SPLIT ? 2 : 1) * Stage::plane, kQDepthMajor, kBK * 128);
                        constexpr uint64_t lo = Stage::plane / 16;
#pragma unroll
                        for (int k = 0; k < kBK / 16; ++k) {
                            mma_pair(d, p + k * 2, q + k * q_step, idesc, s > s0 || k > 0, leader);
                            if (SPLIT) {
                                mma_pair(d, p + k * 2, q + lo + k * q_step, idesc, true, leader);
                                mma_pair(d, p + lo + k * 2, q + k * q_step, idesc, true, leader);
                            }
                        }
                        commit_pair(&sh.empty[stage], leader);
                        if (++stage == kStages) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                    if (!ok) abort_other(abort, rank); // found set by both epilogues behind this barrier
                    commit_pair(&sh.acc_full[acc], leader);
                    issued = true;
                    acc ^= 1;
                    if (acc == 0) acc_phase ^= 1u;
                }
            }
            if (!ok) {
                abort_other(abort, rank);
                const uint32_t last_phase = acc == 0 ? acc_phase ^ 1u : acc_phase; // the products in flight, with a limit
                for (unsigned i = 0; issued && i < kWaitLimit && !mbar_try(&sh.acc_full[acc ^ 1], last_phase); ++i) {}
            }
        }
    }
    } else {
        if (SPLIT) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpilogueRegisters));
        // the epilogue: warp w has rows 32 (w % 4) .., columns W (w / 4) .. of this block's half
        const int row = 32 * (warp % 4) + lane, half = warp / 4;
        float *out_stage = reinterpret_cast<float *>(raw + (stage0 - smem_u32(raw)) + kStages * Stage::bytes) + warp * 32 * kStagePitch;
        const bool poisoned = !E::to_planes && *(volatile const int *)g.error != 0;
        const uint32_t acc_empty[2] = {at_leader(smem_u32(&sh.acc_empty[0])), at_leader(smem_u32(&sh.acc_empty[1]))};
        int acc = 0;
        uint32_t acc_phase = 0;
        bool ok = true;
        for (long long t = first; ok && t < tiles; t += pairs) {
            const TileAt at = tile_at<kBM>(t, per, tiles_n, kSymmetric);
            const int tensor = tab.n > 0 ? muon_tensor_of(tab, at.b) : 0;
            if (tab.n > 0 && !muon_visible(tab, tensor, at.b)) continue;
            const int i = at.i * kPair + (int)rank * 128 + row, j = at.j * kPair + half * W;
            const bool mirror = at.i != at.j;
            Eight e[4];
            float di = 0.f;
            if (E::row_diag && i < g.M) di = g.diag_in[(size_t)at.b * g.M + i];
            fetch32<SPLIT, EPI>(g, at.b, i - lane, j, lane, e);
            auto release = [&] {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) arrive_at(acc_empty[acc]);
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1u;
            };
            auto finish = [&](int c, float *v) {
                const float dj = E::col_diag && j + c + lane < g.N ? g.diag_in[(size_t)at.b * g.M + j + c + lane] : 0.f;
                uint32_t p[32];
                fetch_params<EPI>(g, tab, tensor, at.b, i, j + c, lane, p);
                stage32<SPLIT, EPI>(out_stage, lane, e);
                if (c + 32 < W) fetch32<SPLIT, EPI>(g, at.b, i - lane, j + c + 32, lane, e);
                finish32<SPLIT, EPI>(g, tab, tensor, at.b, i, j + c, lane, v, p, di, dj, mirror, poisoned, out_stage);
            };
            if (SPLIT) { // the sum goes on in registers
                float v[W];
                for (int s0 = 0; ok && s0 < total; s0 += chunk) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&sh.acc_full[acc], acc_phase, abort));
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t src = tmem + ((uint32_t)(32 * (warp % 4)) << 16) + acc * kPair + half * W;
#pragma unroll
                    for (int c = 0; c < W; c += 16) {
                        float u[16];
                        tmem_load16(src + c, u);
#pragma unroll
                        for (int k = 0; k < 16; ++k) v[c + k] = s0 == 0 ? u[k] : v[c + k] + u[k];
                    }
                    release();
                }
                if (!ok) break;
#pragma unroll
                for (int c = 0; c < W; c += 32) finish(c, v + c);
            } else {
                ok = __all_sync(0xffffffffu, mbar_wait(&sh.acc_full[acc], acc_phase, abort));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t src = tmem + ((uint32_t)(32 * (warp % 4)) << 16) + acc * kPair + half * W;
#pragma unroll 1
                for (int c = 0; c < W; c += 32) {
                    float v[32];
                    tmem_load32(src + c, v);
                    finish(c, v);
                }
                release();
            }
        }
    }
    if (warp < kEpilogueWarps && *abort) abort_other(abort, rank);
    if (threadIdx.x == 0 && *abort) atomicExch(g.error, 1);
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_barrier(); // neither block leaves while the other may reach its shared memory
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (!E::to_planes && warp < kEpilogueWarps && *abort) give_up<EPI, kPair, kPair>(g, tab, first, tiles, pairs, per, tiles_n, (int)rank * 128);
    if (warp == kEpilogueWarps + 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * kPair) : "memory");
}

template <bool SPLIT, int EPI>
static int pair_one(const OrthoGemm &g, const GemmMaps &maps, const MuonTable &tab, int per, int tn, long long tiles, int sms,
                    cudaStream_t stream) {
    auto *kernel = ortho_pair_kernel<SPLIT, EPI>;
    constexpr int smem = PairStages<SPLIT>::smem;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
        return check_launch("ortho_pair_kernel attributes");
    if (SPLIT) { // the warpgroups' shares must be what the block is launched with, or they would be waited for
        static std::atomic<int> registers{0}; // 0: not known
        if (registers == 0) {
            cudaFuncAttributes a;
            if (cudaFuncGetAttributes(&a, kernel) != cudaSuccess) return check_launch("ortho_pair_kernel registers");
            registers = a.numRegs;
        }
        if (registers != kPairRegisters) return kPairUnfit;
    }
    const long long pairs = tiles < sms / 2 ? tiles : sms / 2;
    return launch_after(kernel, (unsigned)(2 * pairs), kPairThreads, smem, stream, "ortho_pair_kernel", g, maps, tab, per, tn, tiles);
}

template <bool SPLIT>
int ortho_pair_launch(const OrthoGemm &g, const GemmMaps &maps, const MuonTable &tab, int sms, cudaStream_t stream) {
    const int tm = (g.M + kPair - 1) / kPair, tn = (g.N + kPair - 1) / kPair;
    const int per = g.symmetric ? tm * (tm + 1) / 2 : tm * tn;
    const long long tiles = g.batch * per;
    switch (g.epilogue) {
    case kEpiGram: return pair_one<SPLIT, kEpiGram>(g, maps, tab, per, tn, tiles, sms, stream);
    case kEpiSquare: return pair_one<SPLIT, kEpiSquare>(g, maps, tab, per, tn, tiles, sms, stream);
    case kEpiApply: return pair_one<SPLIT, kEpiApply>(g, maps, tab, per, tn, tiles, sms, stream);
    case kEpiOut: return pair_one<SPLIT, kEpiOut>(g, maps, tab, per, tn, tiles, sms, stream);
    case kEpiMuon: return pair_one<SPLIT, kEpiMuon>(g, maps, tab, per, tn, tiles, sms, stream);
    default: break;
    }
    if constexpr (SPLIT) {
        if (g.epilogue == kEpiSym) return pair_one<SPLIT, kEpiSym>(g, maps, tab, per, tn, tiles, sms, stream);
        return pair_one<SPLIT, kEpiAnti>(g, maps, tab, per, tn, tiles, sms, stream);
    }
    return set_error(kErrUnsupported, "orthogonalize: a backward product of hi planes alone");
}

extern template int ortho_pair_launch<true>(const OrthoGemm &, const GemmMaps &, const MuonTable &, int, cudaStream_t);
extern template int ortho_pair_launch<false>(const OrthoGemm &, const GemmMaps &, const MuonTable &, int, cudaStream_t);

} // namespace gsb
