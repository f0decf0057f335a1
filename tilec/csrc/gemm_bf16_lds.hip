// The tile variants of the bf16 GEMM with direct-to-LDS copies (the kernel:
// gemm_bf16_lds.h) and their launch.
#include "gemm_bf16_lds.h"
#include "../../include/tilec.h"

namespace tilec {

// Launch the LDS-DMA kernel; the caller has checked alignment (16-byte
// operands, contiguous extents and strides multiples of 8) and the 32-bit
// offset limits.
template <int BM, int BN, int BK, int NBUF, int WM, int WN, bool CA, bool CB, int MF>
hipError_t launch_gemm_bf16_lds(const MatmulArgs& a) {
  using P = LdsGemm<BM, BN, BK, NBUF, WM, WN, CA, CB, MF>;
  const int64_t tiles = cdiv(a.M, BM) * cdiv(a.N, BN);
  if (tiles == 0) return hipSuccess;
  const SplitGeom g = gemm_split_geom(a.K, BK, a.split_k);
  if (g.splits > 1 && P::TM * P::TN * P::ACC > kSplitMaxAccPerThread) return hipErrorInvalidConfiguration;
  // The 16x16 pipeline holds more fragment registers; with K % BK != 0 its
  // per-lane K masks no longer fit in 256 VGPRs, so that case runs the 32x32
  // kernel of the same tile.
  if constexpr (MF == 16) {
    if (a.K % BK != 0) return launch_gemm_bf16_lds<BM, BN, BK, NBUF, WM, WN, CA, CB, 32>(a);
  }
  auto kern = gemm_bf16_lds_kernel<BM, BN, BK, NBUF, WM, WN, kKFull, CA, CB, MF, StoreC>;
  if constexpr (MF == 32) {
    if (a.K % BK != 0) kern = gemm_bf16_lds_kernel<BM, BN, BK, NBUF, WM, WN, kKMasked, CA, CB, MF, StoreC>;
  }
  hipLaunchKernelGGL(kern, dim3((unsigned)tiles, (unsigned)g.splits), dim3(P::NT), 0, a.stream,
                     static_cast<const u16*>(a.x1), static_cast<const u16*>(a.x2), StoreC{a.out, a.ldo}, (int)a.M,
                     (int)a.N, (int)a.K, a.ldx1, a.ldx2, 4, device_xcds(), (int)g.steps, g.splits > 1 ? static_cast<float*>(a.workspace) : nullptr,
                     g.splits > 1 ? a.counters : nullptr);
  return hipGetLastError();
}

#define TILEC_LDS_VARIANT(BM, BN, BK, NBUF, WM, WN, MF)                                                \
  template hipError_t launch_gemm_bf16_lds<BM, BN, BK, NBUF, WM, WN, false, false, MF>(const MatmulArgs&); \
  template hipError_t launch_gemm_bf16_lds<BM, BN, BK, NBUF, WM, WN, true, false, MF>(const MatmulArgs&);  \
  template hipError_t launch_gemm_bf16_lds<BM, BN, BK, NBUF, WM, WN, false, true, MF>(const MatmulArgs&);  \
  template hipError_t launch_gemm_bf16_lds<BM, BN, BK, NBUF, WM, WN, true, true, MF>(const MatmulArgs&);
TILEC_LDS_VARIANT(256, 256, 32, 4, 2, 2, 32)
TILEC_LDS_VARIANT(256, 256, 64, 2, 2, 4, 32)
TILEC_LDS_VARIANT(256, 128, 64, 3, 4, 2, 32)
TILEC_LDS_VARIANT(256, 128, 32, 4, 2, 2, 32)
TILEC_LDS_VARIANT(128, 128, 64, 4, 2, 4, 32)
TILEC_LDS_VARIANT(256, 256, 32, 4, 2, 4, 32)
TILEC_LDS_VARIANT(256, 256, 64, 2, 2, 4, 16)
TILEC_LDS_VARIANT(256, 256, 32, 4, 2, 4, 16)
TILEC_LDS_VARIANT(256, 128, 64, 3, 4, 2, 16)
TILEC_LDS_VARIANT(128, 128, 64, 4, 2, 4, 16)
TILEC_LDS_VARIANT(64, 64, 64, 4, 2, 2, 32)
TILEC_LDS_VARIANT(64, 64, 64, 4, 2, 2, 16)
TILEC_LDS_VARIANT(128, 64, 64, 3, 2, 2, 32)
TILEC_LDS_VARIANT(128, 64, 64, 3, 2, 2, 16)
TILEC_LDS_VARIANT(64, 128, 64, 3, 2, 2, 32)
TILEC_LDS_VARIANT(64, 128, 64, 3, 2, 2, 16)
TILEC_LDS_VARIANT(128, 128, 64, 2, 2, 2, 32)
TILEC_LDS_VARIANT(128, 128, 64, 2, 2, 2, 16)
#undef TILEC_LDS_VARIANT

}  // namespace tilec
