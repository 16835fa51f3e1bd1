// gated_norm.h for x of bf16 and a residual of float.
#include "gated_norm.h"

int moc::gn_fwd_bf(const moc_gated_norm& a, bool vec, hipStream_t stream) { return gn::fwd_types<bf16, float>(a, vec, stream); }
int moc::gn_bwd_bf(const moc_gated_norm& a, const moc_gated_norm_grads& g, bool vec, const GnStrips& s, hipStream_t stream) {
  return gn::bwd_types<bf16, float>(a, g, vec, s, stream);
}
