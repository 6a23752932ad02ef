// Layer norm on f32 activations (norm.hpp).
#include "norm.hpp"

namespace mmvae {

int64_t norm_bwd_ws(int64_t M, int64_t N) { return norm_ws_bytes(M, N); }

hipError_t norm_fwd_f32(const mmvae_norm_args& a, hipStream_t st) { return norm_fwd_t<float>(a, st); }
hipError_t norm_bwd_f32(const mmvae_norm_args& a, hipStream_t st) { return norm_bwd_t<float>(a, st); }

}  // namespace mmvae
