// gated_norm.h for x of float and a residual of bf16.
#include "gated_norm.h"

int moc::gn_fwd_fb(const moc_gated_norm& a, bool vec, hipStream_t stream) { return gn::fwd_types<float, bf16>(a, vec, stream); }
int moc::gn_bwd_fb(const moc_gated_norm& a, const moc_gated_norm_grads& g, bool vec, const GnStrips& s, hipStream_t stream) {
  return gn::bwd_types<float, bf16>(a, g, vec, s, stream);
}
