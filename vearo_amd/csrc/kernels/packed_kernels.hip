// packed_kernels.hip -- the second code object that libvearo_hip.so embeds: the
// operators of packed training (query / key norm and rotation, attention over packed
// sequences, cross-entropy of a linear layer). Same conventions as vearo_kernels.hip.
#include "linxent.h"
#include "packed.h"
#include "packed_mm.h"
#include "rope.h"

// Query / key norm and rotation: vh_rope_{fwd,bwd}_v<VW>_l<lanes per row>_n<slots per lane>
#define K_ROPE(VW, L, N)                                                                                            \
  extern "C" __global__ void __launch_bounds__(256) vh_rope_fwd_v##VW##_l##L##_n##N(RopeArgs a) { rope_fwd_impl<VW, L, N>(a); } \
  extern "C" __global__ void __launch_bounds__(256) vh_rope_bwd_v##VW##_l##L##_n##N(RopeArgs a) { rope_bwd_impl<VW, L, N>(a); }
K_ROPE(4, 4, 1) K_ROPE(4, 8, 1) K_ROPE(4, 16, 1) K_ROPE(4, 32, 1) K_ROPE(1, 64, 1) K_ROPE(1, 64, 2)

// Attention over packed sequences, by head size padded to 16 (past 128: to 64). Waves a
// SIMD: what the registers allow. (dk and dv of 80 elements spill 3 registers for the second
// wave: 5003 tokens in 37 sequences, 12 on 6 heads, forward and backward 211 -> 190 us. Of 96
// it would be 25: 8167 tokens, 8 heads, 624 -> 695.)
#define K_PA_LDS(DP)                                                        \
  __shared__ __attribute__((aligned(1024))) uint16_t halves[kPaBwdLds<DP>]; \
  const PaHalves lds = (PaHalves)halves;
#define K_PA(DP, W1, W2, W3, HALVES)                                                                              \
  extern "C" __global__ void __launch_bounds__(256) vh_pa_prep_##DP(PaArgs a) { pa_prep_impl<DP>(a); }               \
  extern "C" __global__ void __launch_bounds__(256, W1) vh_pa_fwd_##DP(PaArgs a) { pa_mm_fwd_impl<DP, 4>(a); }    \
  extern "C" __global__ void __launch_bounds__(256, W2) vh_pa_dq_##DP(PaArgs a) { K_PA_LDS(DP) pa_mm_dq_impl<DP, 4>(a, blockIdx.x, lds); } \
  extern "C" __global__ void __launch_bounds__(256, W3) vh_pa_dkdv_##DP(PaArgs a) { K_PA_LDS(DP) pa_mm_dkdv_impl<DP, 4, HALVES>(a, blockIdx.x, lds); } \
  extern "C" __global__ void __launch_bounds__(256) vh_pa_join_##DP(PaArgs a) { pa_join_impl<DP>(a); } \
  extern "C" __global__ void __launch_bounds__(256) vh_pa_fold_##DP(PaArgs a) { pa_fold_impl<DP>(a); }
K_PA(32, 4, 4, 3, 1) K_PA(48, 3, 3, 2, 1) K_PA(64, 3, 3, 2, 1) K_PA(80, 2, 2, 2, 1) K_PA(96, 2, 2, 1, 1)
K_PA(112, 2, 1, 1, 1) K_PA(128, 2, 1, 1, 1) K_PA(192, 1, 1, 1, 2) K_PA(256, 1, 1, 1, 2)
#define K_PA_BWD(DP, W) \
  extern "C" __global__ void __launch_bounds__(256, W) vh_pa_bwd_##DP(PaArgs a) { K_PA_LDS(DP) pa_mm_bwd_impl<DP, 4>(a, lds); }
K_PA_BWD(32, 3) K_PA_BWD(48, 2) K_PA_BWD(64, 2) K_PA_BWD(80, 2) K_PA_BWD(96, 1) K_PA_BWD(112, 1) K_PA_BWD(128, 1)

// Cross-entropy of a linear layer.
extern "C" __global__ void __launch_bounds__(1024) vh_lx_count(LxCountArgs a) { lx_count_impl(a); }
extern "C" __global__ void __launch_bounds__(LX_BLOCK) vh_lx_stats(LxArgs a) { lx_row_impl<true, false>(a); }
extern "C" __global__ void __launch_bounds__(LX_BLOCK) vh_lx_grad(LxArgs a) { lx_row_impl<false, true>(a); }
extern "C" __global__ void __launch_bounds__(LX_BLOCK) vh_lx_stats_grad(LxArgs a) { lx_row_impl<true, true>(a); }
extern "C" __global__ void __launch_bounds__(1024) vh_lx_loss(LxLossArgs a) { lx_loss_impl(a); }
extern "C" __global__ void __launch_bounds__(256) vh_lx_split(LxSplitArgs a) { lx_split_impl(a); }
extern "C" __global__ void __launch_bounds__(256, 2) vh_lx_logits(LxLogitArgs a) { lx_logits_impl(a); }
extern "C" __global__ void __launch_bounds__(256) vh_lx_finish(LxFinishArgs a) { lx_finish_impl(a); }
extern "C" __global__ void __launch_bounds__(256) vh_lx_tops(LxColsArgs a) { lx_tops_impl(a); }
extern "C" __global__ void __launch_bounds__(512) vh_lx_cols(LxColsArgs a) { lx_cols_impl(a); }
extern "C" __global__ void __launch_bounds__(512) vh_lx_dz(LxDzArgs a) { lx_dz_impl(a); }
extern "C" __global__ void __launch_bounds__(256, 2) vh_lx_mm(LxMmArgs a) { lx_mm_impl(a); }
extern "C" __global__ void __launch_bounds__(256) vh_lx_join(LxMmArgs a) { lx_join_impl(a); }
