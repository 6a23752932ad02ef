// The layer operators' launchers (ops.hip), shared by their C entries and the wide path.  The
// arguments are checked by *_check (null: fine); the launchers trust them.
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/mmvae_capi.h"

namespace mmvae {

hipError_t norm_fwd(const mmvae_norm_args& a, hipStream_t st);
hipError_t norm_bwd(const mmvae_norm_args& a, hipStream_t st);
int64_t norm_bwd_ws(int64_t M, int64_t N);
// one type each (norm_f32 / _bf16 / _f16.hip; M > 0)
hipError_t norm_fwd_f32(const mmvae_norm_args& a, hipStream_t st);
hipError_t norm_bwd_f32(const mmvae_norm_args& a, hipStream_t st);
hipError_t norm_fwd_bf16(const mmvae_norm_args& a, hipStream_t st);
hipError_t norm_bwd_bf16(const mmvae_norm_args& a, hipStream_t st);
hipError_t norm_fwd_f16(const mmvae_norm_args& a, hipStream_t st);
hipError_t norm_bwd_f16(const mmvae_norm_args& a, hipStream_t st);
hipError_t dropout(const mmvae_dropout_args& a, hipStream_t st);
hipError_t emb_fwd(const mmvae_embedding_args& a, hipStream_t st);
hipError_t emb_bwd(const mmvae_embedding_args& a, hipStream_t st);
int64_t emb_bwd_ws(int64_t T, int64_t N, int64_t V);
const char* norm_check(const mmvae_norm_args& a, bool bwd);
const char* dropout_check(const mmvae_dropout_args& a);
const char* emb_check(const mmvae_embedding_args& a, bool bwd);

// the calling thread's message for mmvae_last_error(NULL); returns `code` (capi.hip)
int set_last_error(int code, const char* op, const char* msg) noexcept;

}  // namespace mmvae
