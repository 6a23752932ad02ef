// Device helpers of the layer operators (ops.hip, norm.hpp): chunks of 8 elements, lane sums, dropout
// masks, and the kernel launch.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <tuple>
#include <type_traits>
#include <utility>

#include "common.hpp"
#include "ops.hpp"

namespace mmvae {

// =======================================================================================
// Chunks: 8 consecutive elements
// =======================================================================================
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef _Float16 f16x8u __attribute__((ext_vector_type(8), aligned(2)));

template <class T> struct Chunk;
template <> struct Chunk<float> {
    f32x4u a, b;
    MMVAE_DEV float get(int i) const { return i < 4 ? a[i & 3] : b[i & 3]; }
    MMVAE_DEV void set(int i, float v) {
        if (i < 4) a[i & 3] = v;
        else b[i & 3] = v;
    }
    static MMVAE_DEV Chunk load(const float* p) {
        return Chunk{*reinterpret_cast<const f32x4u*>(p), *reinterpret_cast<const f32x4u*>(p + 4)};
    }
    MMVAE_DEV void store(float* p) const {
        *reinterpret_cast<f32x4u*>(p) = a;
        *reinterpret_cast<f32x4u*>(p + 4) = b;
    }
    MMVAE_DEV void anew() { asm("" : "+v"(a), "+v"(b)); }  // (what was computed from it is computed again, not kept)
    MMVAE_DEV void keep(const bool on[8]) {                // the others: 0
#pragma unroll
        for (int i = 0; i < 8; ++i) set(i, on[i] ? get(i) : 0.f);
    }
};
template <class T, class V> struct Chunk16 {
    V v;
    MMVAE_DEV float get(int i) const { return (float)v[i]; }
    MMVAE_DEV void set(int i, float x) { v[i] = (T)x; }  // to nearest even
    MMVAE_DEV void anew() { asm("" : "+v"(v)); }
    MMVAE_DEV void keep(const bool on[8]) {
        typedef uint32_t u4 __attribute__((ext_vector_type(4)));
        u4 w = __builtin_bit_cast(u4, v);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] &= (on[2 * k] ? 0xffffu : 0u) | (on[2 * k + 1] ? 0xffff0000u : 0u);
        v = __builtin_bit_cast(V, w);
    }
};
template <> struct Chunk<__bf16> : Chunk16<__bf16, bf16x8u> {
    static MMVAE_DEV Chunk load(const __bf16* p) {
        Chunk c;
        c.v = *reinterpret_cast<const bf16x8u*>(p);
        return c;
    }
    MMVAE_DEV void store(__bf16* p) const { *reinterpret_cast<bf16x8u*>(p) = v; }
};
template <> struct Chunk<_Float16> : Chunk16<_Float16, f16x8u> {
    static MMVAE_DEV Chunk load(const _Float16* p) {
        Chunk c;
        c.v = *reinterpret_cast<const f16x8u*>(p);
        return c;
    }
    MMVAE_DEV void store(_Float16* p) const { *reinterpret_cast<f16x8u*>(p) = v; }
};

// The n valid elements of a chunk (n <= 0: none), zeros behind them.  A row's last chunk (n < 8) goes
// in the pieces of n's binary digits: 4, 2 and 1 elements, three accesses however many.
typedef float f32x2u __attribute__((ext_vector_type(2), aligned(4)));
typedef uint32_t u32x2u __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(2))) u32u {
    uint32_t v;
};
MMVAE_DEV Chunk<float> ld_tail(const float* p, int n) {
    float q0 = 0.f, q1 = 0.f, q2 = 0.f, q3 = 0.f, d0 = 0.f, d1 = 0.f, h = 0.f;
    const bool n4 = n & 4, n2 = n & 2;
    if (n4) {
        const f32x4u q = *reinterpret_cast<const f32x4u*>(p);
        q0 = q[0]; q1 = q[1]; q2 = q[2]; q3 = q[3];
    }
    if (n2) {
        const f32x2u d = *reinterpret_cast<const f32x2u*>(p + (n & 4));
        d0 = d[0]; d1 = d[1];
    }
    if (n & 1) h = p[n & 6];
    const float r0 = n2 ? d0 : h, r2 = n2 ? h : 0.f;
    Chunk<float> c;
    c.a[0] = n4 ? q0 : r0; c.a[1] = n4 ? q1 : d1; c.a[2] = n4 ? q2 : r2; c.a[3] = n4 ? q3 : 0.f;
    c.b[0] = n4 ? r0 : 0.f; c.b[1] = n4 ? d1 : 0.f; c.b[2] = n4 ? r2 : 0.f; c.b[3] = 0.f;
    return c;
}
template <class T> MMVAE_DEV Chunk<T> ld_tail(const T* p, int n) {  // 16-bit elements
    uint32_t q0 = 0, q1 = 0, d = 0, h = 0;
    const bool n4 = n & 4, n2 = n & 2;
    if (n4) {
        const u32x2u q = *reinterpret_cast<const u32x2u*>(p);
        q0 = q[0];
        q1 = q[1];
    }
    if (n2) d = reinterpret_cast<const u32u*>(p + (n & 4))->v;
    if (n & 1) h = reinterpret_cast<const uint16_t*>(p)[n & 6];
    const uint32_t lo = n2 ? d : h, hi = n2 ? h : 0;
    const u32x4 r = {n4 ? q0 : lo, n4 ? q1 : hi, n4 ? lo : 0, n4 ? hi : 0};
    Chunk<T> c;
    c.v = __builtin_bit_cast(decltype(c.v), r);
    return c;
}
template <class T> MMVAE_DEV Chunk<T> ld8(const T* p, int n) {
    if (n >= 8) return Chunk<T>::load(p);
    return ld_tail(p, n > 0 ? n : 0);
}
MMVAE_DEV void st_tail(float* p, int n, const Chunk<float>& c) {
    const bool n4 = n & 4;
    if (n4) *reinterpret_cast<f32x4u*>(p) = c.a;
    const float r0 = n4 ? c.b[0] : c.a[0], r1 = n4 ? c.b[1] : c.a[1], r2 = n4 ? c.b[2] : c.a[2];
    if (n & 2) *reinterpret_cast<f32x2u*>(p + (n & 4)) = f32x2u{r0, r1};
    if (n & 1) p[n & 6] = (n & 2) ? r2 : r0;
}
template <class T> MMVAE_DEV void st_tail(T* p, int n, const Chunk<T>& c) {
    const u32x4 v = __builtin_bit_cast(u32x4, c.v);
    const bool n4 = n & 4;
    if (n4) *reinterpret_cast<u32x2u*>(p) = u32x2u{v[0], v[1]};
    const uint32_t r0 = n4 ? v[2] : v[0], r1 = n4 ? v[3] : v[1];
    if (n & 2) reinterpret_cast<u32u*>(p + (n & 4))->v = r0;
    if (n & 1) reinterpret_cast<uint16_t*>(p)[n & 6] = (uint16_t)((n & 2) ? r1 : r0);
}
template <class T> MMVAE_DEV void st8(T* p, int n, const Chunk<T>& c) {
    if (n >= 8) c.store(p);
    else if (n > 0) st_tail(p, n, c);
}
// Chunk col of a row of N.  EVEN (N a multiple of 8): no branch; a lane behind the row's end reads the
// row's first chunk, for the caller to ignore.
template <bool EVEN, class T> MMVAE_DEV Chunk<T> ld_row(const T* row, int col, int N) {
    if constexpr (EVEN) return Chunk<T>::load(row + (col < N ? col : 0));
    else return ld8(row + col, N - col);
}
// a thread's 8 floats in LDS, slot of `slots` (two 16-byte planes: no bank conflicts)
MMVAE_DEV void lds_put8(float* l, int slots, int slot, const float v[8]) {
    *reinterpret_cast<float4*>(l + slot * 4) = float4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<float4*>(l + (slots + slot) * 4) = float4{v[4], v[5], v[6], v[7]};
}
MMVAE_DEV void lds_get8(const float* l, int slots, int slot, float v[8]) {
    const float4 a = *reinterpret_cast<const float4*>(l + slot * 4), b = *reinterpret_cast<const float4*>(l + (slots + slot) * 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
// 8 weights of type T or f32 (w null: `none`)
template <class T> MMVAE_DEV void ldw(const void* w, bool f32, int col, int n, float none, float v[8]) {
    if (!w) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = none;
    } else if (f32) {
        const Chunk<float> c = ld8((const float*)w + col, n);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c.get(i);
    } else {
        const Chunk<T> c = ld8((const T*)w + col, n);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c.get(i);
    }
}

// =======================================================================================
// Sums over the TPR lanes of a row (every lane gets the sum), in registers: DPP within 16 lanes,
// then the two lane swaps
// =======================================================================================
template <int CTRL> MMVAE_DEV float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int TPR> MMVAE_DEV float lanes_sum(float v) {
    v = dpp_add<0xB1>(v);                        // quad_perm [1, 0, 3, 2]
    v = dpp_add<0x4E>(v);                        // quad_perm [2, 3, 0, 1]
    v = dpp_add<0x141>(v);                       // row_half_mirror: the other quad of 8 lanes
    if constexpr (TPR >= 16) v = dpp_add<0x140>(v);  // row_mirror: the other 8 of 16 lanes
    if constexpr (TPR >= 32) {
        const unsigned u = __builtin_bit_cast(unsigned, v);
        const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        v = __builtin_bit_cast(float, (unsigned)s[0]) + __builtin_bit_cast(float, (unsigned)s[1]);
    }
    if constexpr (TPR >= 64) {
        const unsigned u = __builtin_bit_cast(unsigned, v);
        const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        v = __builtin_bit_cast(float, (unsigned)s[0]) + __builtin_bit_cast(float, (unsigned)s[1]);
    }
    return v;
}
// the same over a row's TPR > 64 threads (one row per workgroup): the waves' sums through `red`
template <int TPR> MMVAE_DEV float row_sum(float v, float* red) {
    v = lanes_sum<(TPR < 64 ? TPR : 64)>(v);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < TPR / 64; ++w) v += red[w];
    }
    return v;
}

// =======================================================================================
// Dropout factors.  16 random bits per element: half (col % 8) of the four words of
// Philox4x32-10 at the counter (col / 8, row, step, step >> 32 ^ row >> 32), keyed by the seed;
// kept iff they are >= thr = round(65536 p), so P(kept) = 1 - thr / 65536 exactly and the factor
// 65536 / (65536 - thr) leaves the mean unchanged.  The row is global (row_offset + r), so the
// shards of a data-parallel batch drop what the whole batch would; the mask is never stored: the
// backward recomputes it.  Cost: 20 32 x 32-bit products per 8 elements.
// =======================================================================================
// A dropped element is 0 whatever it was (an infinity or NaN times a factor 0 would be NaN).
struct DropKey {
    uint32_t thr;  // 0: no dropout
    float s;       // the factor of the kept
    uint32_t k0, k1;
    int64_t step, row0;
    const int64_t* state;
};
MMVAE_DEV void drop_state(DropKey& k) {
    if (k.state) {
        k.step += k.state[0];
        k.row0 += k.state[1];
    }
}
// the 8 elements of a chunk that are kept.  (h >= thr on whole words: the high half as it is, the low
// half shifted up; p = 1, thr = 65536, keeps none)
MMVAE_DEV void keep8(const DropKey& k, int64_t row, int chunk, bool kept[8]) {
    const uint64_t r = (uint64_t)(k.row0 + row);
    uint32_t ch = (uint32_t)chunk;
    asm volatile("" : "+v"(ch));  // (a chunk's first products, the same for every row, are not worth their registers)
    uint32_t c0 = ch, c1 = (uint32_t)r, c2 = (uint32_t)k.step, c3 = (uint32_t)((uint64_t)k.step >> 32) ^ (uint32_t)(r >> 32);
    uint32_t k0 = k.k0, k1 = k.k1;
#pragma unroll
    for (int i = 0; i < 10; ++i) {  // (common.hpp's rounds, each three-way xor in one instruction)
        const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
        c0 = __builtin_amdgcn_bitop3_b32((uint32_t)(p1 >> 32), c1, k0, 0x96);
        c2 = __builtin_amdgcn_bitop3_b32((uint32_t)(p0 >> 32), c3, k1, 0x96);
        c1 = (uint32_t)p1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    const uint32_t c[4] = {c0, c1, c2, c3};
    const uint32_t t = k.thr << 16;
    const bool some = k.thr < 65536;
#pragma unroll
    for (int i = 0; i < 8; ++i) kept[i] = ((i & 1) ? c[i >> 1] : c[i >> 1] << 16) >= t && some;
}

// =======================================================================================
// Host side
// =======================================================================================
template <class... P, class... A>
inline hipError_t launch_lds(size_t lds, void (*k)(P...), dim3 grid, dim3 block, hipStream_t st, A&&... args) {
    // the launch's own error (hipGetLastError could return an earlier call's)
    std::tuple<P...> v{static_cast<P>(args)...};
    return std::apply(
        [&](P&... p) {
            void* ptr[] = {(void*)&p...};
            return hipLaunchKernel((const void*)k, grid, block, ptr, lds, st);
        },
        v);
}
template <class... P, class... A>
inline hipError_t launch(void (*k)(P...), dim3 grid, dim3 block, hipStream_t st, A&&... args) {
    return launch_lds(0, k, grid, block, st, std::forward<A>(args)...);
}
#define OPCHK(x)                            \
    do {                                    \
        const hipError_t er_ = (x);         \
        if (er_ != hipSuccess) return er_;  \
    } while (0)

inline uint32_t drop_thr(double p) { return (uint32_t)std::floor(p * 65536. + 0.5); }
inline DropKey drop_key(double p, uint64_t seed, uint64_t step, uint64_t row_offset, const int64_t* state) {
    DropKey k;
    k.thr = drop_thr(p);
    k.s = k.thr < 65536 ? (float)(65536. / (65536. - k.thr)) : 0.f;
    k.k0 = (uint32_t)seed;
    k.k1 = (uint32_t)(seed >> 32);
    k.step = (int64_t)step;
    k.row0 = (int64_t)row_offset;
    k.state = state;
    return k;
}
template <class F> inline hipError_t by_type(int dtype, F&& f) {
    if (dtype == MMVAE_T_F32) return f(float{});
    if (dtype == MMVAE_T_BF16) return f(__bf16{});
    return f(_Float16{});
}
template <int V> using I = std::integral_constant<int, V>;

}  // namespace mmvae
