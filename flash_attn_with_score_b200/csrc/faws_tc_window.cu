// The forward launches of attention_with_window(): the forward kernel's instances whose rows see their last keys and the
// first ones only.
#include <cuda.h>

#include "faws_tc_fwd.cuh"

namespace faws {
namespace {

template <typename T, int D>
cudaError_t launch_t(const TcMaps& maps, const FwdParams& p, cudaStream_t s) {
  if (p.pack_m > 0 || p.n_splits > 1) return launch_fwd_s<T, D, kHookNone, true, kNoDrop, true, true>(maps, p, s);
  // 256-row CTAs, of two heads' rows where the group has an even number of them, against 128-row ones by the times that plain
  // launches of as many key tiles are expected to take.  Over 216 bf16 shapes (D 64 and 128; heads 12-12, 16-4, 28-4, 32-8, 8-1, 14-2; 512
  // to 8192 rows, batches of 1 to 4; windows 64 to 1024; 0, 4, 300 sinks) that is 0.4 % longer than the better of the two, 8 % at
  // the worst, where 256 rows throughout are 8 % longer and 128 rows twice as long; two heads to a CTA are 7.6 % shorter over the 108
  // shapes with even groups, 2.6 % longer at the worst.
  FwdParams pp = p;
  pp.pair_heads = p.G % 2 == 0 ? 1 : 0;
  RowChoice c{(long long)p.B * p.Hq, p.m_begin, p.m_end, p.N, p.p_seq, p.causal, sm_count(), p.window, p.sinks};
  const double small = expected_us(c, D == 128, kPlainOut, 128);
  if (pp.pair_heads) c.heads /= 2;
  const bool large = c.blocks(pp.pair_heads ? 128 : 256) * c.heads >= 2LL * c.sms ||
                     small > 1.03 * expected_us(c, D == 128, kPlainOut, 256, pp.pair_heads ? 128 : 0);
  return large ? launch_fwd_s<T, D, kHookNone, false, kNoDrop, false, true>(maps, pp, s)
               : launch_fwd_s<T, D, kHookNone, true, kNoDrop, false, true>(maps, p, s);
}

}  // namespace

cudaError_t launch_tc_fwd_window(const FwdParams& p, int dtype, cudaStream_t s) {
  TcMaps maps;
  if (!make_fwd_maps(&maps, p)) return cudaErrorInvalidValue;
  if (dtype == FAWS_FP16) return p.D == 128 ? launch_t<__half, 128>(maps, p, s) : launch_t<__half, 64>(maps, p, s);
  return p.D == 128 ? launch_t<__nv_bfloat16, 128>(maps, p, s) : launch_t<__nv_bfloat16, 64>(maps, p, s);
}

}  // namespace faws
