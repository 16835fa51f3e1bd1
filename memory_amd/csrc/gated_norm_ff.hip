// gated_norm.h for x of float and a residual of float.
#include "gated_norm.h"

int moc::gn_fwd_ff(const moc_gated_norm& a, bool vec, hipStream_t stream) { return gn::fwd_types<float, float>(a, vec, stream); }
int moc::gn_bwd_ff(const moc_gated_norm& a, const moc_gated_norm_grads& g, bool vec, const GnStrips& s, hipStream_t stream) {
  return gn::bwd_types<float, float>(a, g, vec, s, stream);
}
