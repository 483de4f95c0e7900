#include "ortho_gemm_pair.cuh"

namespace gsb {
template int ortho_pair_launch<false>(const OrthoGemm &, const GemmMaps &, const MuonTable &, int, cudaStream_t);
} // namespace gsb
