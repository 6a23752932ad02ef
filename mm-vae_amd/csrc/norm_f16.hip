// Layer norm on f16 activations (norm.hpp).
#include "norm.hpp"

namespace mmvae {

hipError_t norm_fwd_f16(const mmvae_norm_args& a, hipStream_t st) { return norm_fwd_t<_Float16>(a, st); }
hipError_t norm_bwd_f16(const mmvae_norm_args& a, hipStream_t st) { return norm_bwd_t<_Float16>(a, st); }

}  // namespace mmvae
