#include "ortho_gemm.cuh"

namespace gsb {
template int ortho_gemm_launch<true, 128>(const OrthoGemm &, const GemmMaps &, const MuonTable &, int, cudaStream_t);
} // namespace gsb
