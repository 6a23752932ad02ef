// Layer norm on bf16 activations (norm.hpp).
#include "norm.hpp"

namespace mmvae {

hipError_t norm_fwd_bf16(const mmvae_norm_args& a, hipStream_t st) { return norm_fwd_t<__bf16>(a, st); }
hipError_t norm_bwd_bf16(const mmvae_norm_args& a, hipStream_t st) { return norm_bwd_t<__bf16>(a, st); }

}  // namespace mmvae
