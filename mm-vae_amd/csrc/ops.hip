// Layer operators on device tensors (mmvae_layer_norm_*, mmvae_dropout, mmvae_embedding_*): the
// normalised, dropped-out, label-conditioned layer chain of the wide path (wide.hip), and the
// same for callers with tensors of their own.  The norm's kernels: norm.hpp.
//
// Every kernel moves 8 consecutive elements per lane ("a chunk": 16 B of bf16 / f16, 32 B of f32),
// which is also what one Philox call masks.  Chunks are loaded at the elements' own alignment, so
// odd widths and row strides take the same path; a row's last, partial chunk goes in pieces.
// Sums, statistics and accumulators are f32; a value is rounded to its type once, when it is
// stored.  Every reduction has a fixed order, so equal calls give equal bits.
#include "ops_dev.hpp"

namespace mmvae {

// =======================================================================================
// Chunks of many rows, dealt out evenly whatever the width: chunk i of all is chunk i % nc of row
// i / nc.  A workgroup takes 1024 in a row, four a thread (their loads in flight together); the
// division is once per workgroup, and within it by a float product (li + 1/2) / nc, whose distance
// from a whole number, >= 1 / (2 nc), is above its error for li < 2^22 (N < 2^24, or one row's part).
// =======================================================================================
static constexpr int WALK = 4;
struct Walk {
    int64_t row0;  // the workgroup's first chunk: its row and place there
    int c0;
    float inv;
    int nc;
};
MMVAE_DEV Walk walk_from(int64_t nc) {
    const int64_t i = (int64_t)blockIdx.x * (256 * WALK), r = i / nc;
    return Walk{r, (int)(i - r * nc), 1.f / (float)nc, (int)nc};
}
MMVAE_DEV int64_t walk_row(const Walk& w, int u, int* chunk) {
    const int li = w.c0 + u * 256 + (int)threadIdx.x, q = (int)(((float)li + 0.5f) * w.inv);
    *chunk = li - q * w.nc;
    return w.row0 + q;
}
static int64_t walk_blocks(int64_t rows, int64_t N) { return (rows * ((N + 7) / 8) + 256 * WALK - 1) / (256 * WALK); }

// =======================================================================================
// Dropout alone.  Bound by memory: 4096 x 20000 bf16 (328 MB) 58 us, 5.6 TB/s (part of the input comes from
// the last-level cache); the mask's 20 products for 8 elements stay below the loads' time, its four chunks a
// thread in flight are what the rate needs (one row a workgroup, as it was first, 66 us).
// =======================================================================================
template <class T>
__global__ __launch_bounds__(256) void k_dropout(int64_t M, int N, const T* x, int64_t ldx, T* y, int64_t ldy, DropKey k) {
    drop_state(k);
    const Walk w = walk_from((N + 7) / 8);
    int c[WALK];
    int64_t row[WALK];
    Chunk<T> v[WALK];
#pragma unroll
    for (int u = 0; u < WALK; ++u) {
        row[u] = walk_row(w, u, &c[u]);
        v[u] = ld8(x + (row[u] < M ? row[u] : 0) * ldx + c[u] * 8, N - c[u] * 8);
    }
#pragma unroll
    for (int u = 0; u < WALK; ++u) {
        if (row[u] >= M) break;
        bool kept[8];
        keep8(k, row[u], c[u], kept);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u].set(i, kept[i] ? v[u].get(i) * k.s : 0.f);
        st8(y + row[u] * ldy + c[u] * 8, N - c[u] * 8, v[u]);
    }
}

// =======================================================================================
// Embedding: y[t] = scale table[id_t] (+ add[t]), zero rows for ids outside [0, V).  Bound by the rows
// written and the table rows read, of which hot ones come from L2: 262144 x 128 bf16 16 us (67 MB written,
// 4.2 TB/s), 50001 x 517 f16 19 us (52 MB).
// =======================================================================================
struct EmbF {
    int64_t T;
    int N;
    int64_t V;
    const void *ids, *table, *add;
    int64_t ldt, ldadd, ldy;
    void* y;
    float scale;
    int i64;
};
MMVAE_DEV int64_t emb_id(const void* ids, int i64, int64_t t) {
    return i64 ? ((const int64_t*)ids)[t] : (int64_t)((const int32_t*)ids)[t];
}
template <class T> __global__ __launch_bounds__(256) void k_emb_fwd(EmbF a) {
    const Walk w = walk_from((a.N + 7) / 8);
    int c[WALK];
    int64_t t[WALK], id[WALK];
    Chunk<T> v[WALK];
#pragma unroll
    for (int u = 0; u < WALK; ++u) {
        t[u] = walk_row(w, u, &c[u]);
        id[u] = emb_id(a.ids, a.i64, t[u] < a.T ? t[u] : 0);
    }
#pragma unroll
    for (int u = 0; u < WALK; ++u) {
        const bool ok = id[u] >= 0 && id[u] < a.V;
        v[u] = ld8((const T*)a.table + (ok ? id[u] : 0) * a.ldt + c[u] * 8, ok ? a.N - c[u] * 8 : 0);
    }
#pragma unroll
    for (int u = 0; u < WALK; ++u) {
        if (t[u] >= a.T) break;
        const bool ok = id[u] >= 0 && id[u] < a.V;
        const int col = c[u] * 8, n = a.N - col;
        if (a.add) {
            const Chunk<T> d = ld8((const T*)a.add + t[u] * a.ldadd + col, n);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[u].set(i, ok ? __builtin_fmaf(v[u].get(i), a.scale, d.get(i)) : d.get(i));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[u].set(i, ok ? v[u].get(i) * a.scale : 0.f);
        }
        st8((T*)a.y + t[u] * a.ldy + col, n, v[u]);
    }
}

// =======================================================================================
// Embedding gradient: dE[v] = scale sum over the tokens of v of dy.
// Many table rows (V > FEW):
//   1. the tokens sorted by id, stable (LSD radix sort, 8-bit digits; ids outside [0, V) as V,
//      behind all others): in one workgroup up to 4096 tokens, else histogram + scatter per digit;
//   2. k_emb_seg: fixed pieces of the sorted tokens, whatever their ids: a hot id is spread over
//      many workgroups, the sums of runs inside a piece are final, the first and last run of a
//      piece leave a partial where they go on in the next one;
//   3. k_emb_join: the partials of a run that crosses pieces, summed in order.
// Few rows (labels: V <= FEW), where a sort of all tokens would cost more than their sums: each
// piece sorts its own tokens and leaves one partial per row it has (k_emb_seg<FEW>), and
// k_emb_few_join adds them up in order.
// No atomics on sums: equal calls give equal bits.  dy is read once; what is left beside it is the sort,
// a chain of short kernels.  262144 tokens into 20000 x 128 bf16: histograms 4.4 + 3.9 us, scatters 2 x 7.5,
// k_emb_seg 15.8 (67 MB of dy, 4.2 TB/s), k_emb_join 4.3.  50001 into 30011 x 517 f16: 6.6 (with the 31 MB
// of zeros) + 3.6, 2 x 6.7, 23.4 (52 MB in rows that end inside a cache line), 4.8.  4096 labels into 12 x
// 128 f32: 5.8 + 3.4.
// =======================================================================================
static constexpr int FEW = 64;      // (128 columns bf16, 64 rows against 65 sorted: 256 tokens 8.2 / 12.2 us, 4096
                                    // 8.9 / 15.3, 32768 16.2 / 18.3, 262144 30.5 / 28.9: level from there, whatever T)
static constexpr int RTHR = 1024;   // a sort tile: 16 waves x KPT x 64 tokens
static constexpr int RONE = 4096;   // tokens that one workgroup sorts, KPT = 4 (4096 tokens into 20000 x 128 bf16
                                    // 19.4 us, 4097 in tiles 24.9)
static constexpr int RTILE = 2048;  // a tile of a longer sort, KPT = 2 (a scatter of 262144 tokens 7.5 us, with tiles of
                                    // 1024 or 4096 9.2; of 50001 tokens 6.7, 1024 5.9, 4096 8.6)
static constexpr int RFUSE = 256;   // up to so many tiles a scatter workgroup sums the histograms itself: a
                                    // launch less (64 columns: 524288 tokens 47.4 us, one more 51.7)

// Stable ranks of the workgroup's keys by an 8-bit digit (16 waves, KPT keys a lane; wave w holds the
// tokens w 64 KPT + k 64 + lane).  wh[w][d]: first the wave's counts, then the count of d in earlier waves.
struct RadixLds {
    uint32_t wh[RTHR / 64][256];
    uint32_t tot[2][256];   // the tile's count of each digit; all tiles'
    uint32_t base[2][256];  // exclusive sums of the two
    uint32_t ws[8];
};
template <int RKPT> MMVAE_DEV void radix_rank(const uint32_t dig[RKPT], const bool val[RKPT], uint32_t rank[RKPT], RadixLds& L) {
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int i = threadIdx.x; i < (RTHR / 64) * 256; i += RTHR) L.wh[i >> 8][i & 255] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < RKPT; ++k) {
        const uint32_t old = val[k] ? L.wh[w][dig[k]] : 0;  // (comes while the lanes of the same digit are found)
        const uint64_t valid = __ballot(val[k]);
        uint32_t m0 = (uint32_t)valid, m1 = (uint32_t)(valid >> 32);
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const uint32_t bit = (uint32_t)((int32_t)(dig[k] << (31 - b)) >> 31);  // 0 or all ones
            const uint64_t bal = __ballot(bit != 0);
            m0 &= ~((uint32_t)bal ^ bit);
            m1 &= ~((uint32_t)(bal >> 32) ^ bit);
        }
        const uint32_t lt = __builtin_amdgcn_mbcnt_hi(m1, __builtin_amdgcn_mbcnt_lo(m0, 0));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (val[k] && lt == 0) L.wh[w][dig[k]] = old + __popc(m0) + __popc(m1);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        rank[k] = old + lt;
    }
    __syncthreads();
    if (threadIdx.x < 256) {
        uint32_t t = 0;
        uint32_t c[RTHR / 64];
#pragma unroll
        for (int q = 0; q < RTHR / 64; ++q) c[q] = L.wh[q][threadIdx.x];
#pragma unroll
        for (int q = 0; q < RTHR / 64; ++q) {
            L.wh[q][threadIdx.x] = t;
            t += c[q];
        }
        L.tot[0][threadIdx.x] = t;
    }
    __syncthreads();
}
// base[k][d] = sum of tot[k][e] over e < d (waves 0 .. 3 the first, 4 .. 7 the second)
MMVAE_DEV void digit_scan(RadixLds& L) {
    const int k = threadIdx.x >> 8, d = threadIdx.x & 255;
    uint32_t own = 0, v = 0;
    if (k < 2) {
        own = v = L.tot[k][d];
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t u = __shfl_up(v, o, 64);
            if ((d & 63) >= o) v += u;
        }
        if ((d & 63) == 63) L.ws[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    if (k < 2) {
        uint32_t b = v - own;
        for (int q = 0; q < (d >> 6); ++q) b += L.ws[4 * k + q];
        L.base[k][d] = b;
    }
    __syncthreads();
}
MMVAE_DEV uint32_t emb_key(const void* ids, int i64, int64_t t, uint32_t V) {
    const int64_t id = emb_id(ids, i64, t);
    return id >= 0 && id < (int64_t)V ? (uint32_t)id : V;
}
// bytes of zeros (out 4-byte aligned), by thread i of `step`
MMVAE_DEV void fill_zero(void* out, int64_t bytes, int64_t i, int64_t step) {
    const int64_t head = ((16 - ((uintptr_t)out & 15)) & 15) < bytes ? (16 - ((uintptr_t)out & 15)) & 15 : bytes;
    uint4* q = reinterpret_cast<uint4*>((char*)out + head);
    const int64_t n = (bytes - head) / 16, rest = bytes - head - n * 16;
    if (i < head / 4) ((uint32_t*)out)[i] = 0;
    if (i < rest / 2) ((uint16_t*)(q + n))[i] = 0;
    if (i == 0 && (head & 2)) ((uint16_t*)out)[head / 2 - 1] = 0;  // (a buffer that ends before its first 16 bytes)
    for (; i < n; i += step) q[i] = make_uint4(0, 0, 0, 0);
}

// the whole sort of T <= RONE tokens in workgroup 0, the keys in registers from pass to pass (a chain of LDS
// round trips: 10 us for two digits of 4096 tokens, 6 for one); the others clear the gradient
__global__ __launch_bounds__(RTHR) void k_emb_sort1(const void* ids, int i64, int T, uint32_t V, int passes, uint2* kv, void* out,
                                                    int64_t out_bytes) {
    if (blockIdx.x > 0) {
        fill_zero(out, out_bytes, (int64_t)(blockIdx.x - 1) * RTHR + threadIdx.x, (int64_t)(gridDim.x - 1) * RTHR);
        return;
    }
    constexpr int KPT = RONE / RTHR;
    __shared__ RadixLds L;
    __shared__ uint2 sh[RONE];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    uint32_t kk[KPT], ii[KPT], dig[KPT], rank[KPT];
    bool val[KPT];
#pragma unroll
    for (int k = 0; k < KPT; ++k) {
        const int t = (w * KPT + k) * 64 + lane;
        val[k] = t < T;
        kk[k] = val[k] ? emb_key(ids, i64, t, V) : 0;
        ii[k] = t;
    }
    for (int p = 0; p < passes; ++p) {
#pragma unroll
        for (int k = 0; k < KPT; ++k) dig[k] = (kk[k] >> (8 * p)) & 255;
        radix_rank<KPT>(dig, val, rank, L);
        digit_scan(L);
#pragma unroll
        for (int k = 0; k < KPT; ++k)
            if (val[k]) sh[L.base[0][dig[k]] + L.wh[w][dig[k]] + rank[k]] = make_uint2(kk[k], ii[k]);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < KPT; ++k) {
            const int t = (w * KPT + k) * 64 + lane;
            if (t < T) {
                kk[k] = sh[t].x;
                ii[k] = sh[t].y;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < KPT; ++k) {
        const int t = (w * KPT + k) * 64 + lane;
        if (t < T) kv[t] = make_uint2(kk[k], ii[k]);
    }
}

// digit counts of each tile, two 16-bit ones a word (digits d and d + 128): hist[tile][128]; kv null: the
// first pass, from the ids.  Workgroups past the tiles (first pass) clear the gradient.
__global__ __launch_bounds__(RTHR) void k_emb_hist(const void* ids, int i64, const uint2* kv, int64_t T, uint32_t V, int shift, int tiles,
                                                   uint32_t* hist, void* out, int64_t out_bytes) {
    if ((int)blockIdx.x >= tiles) {
        const int b = blockIdx.x - tiles, nb = gridDim.x - tiles;
        fill_zero(out, out_bytes, (int64_t)b * RTHR + threadIdx.x, (int64_t)nb * RTHR);
        return;
    }
    __shared__ uint32_t h[256];
    if (threadIdx.x < 256) h[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < RTILE / RTHR; ++k) {
        const int64_t t = (int64_t)blockIdx.x * RTILE + k * RTHR + threadIdx.x;
        if (t < T) atomicAdd(&h[((kv ? kv[t].x : emb_key(ids, i64, t, V)) >> shift) & 255], 1u);
    }
    __syncthreads();
    if (threadIdx.x < 128) hist[(int64_t)blockIdx.x * 128 + threadIdx.x] = h[threadIdx.x] | h[threadIdx.x + 128] << 16;
}
// many tiles: before[tile][d] = the count of d in earlier tiles, before[tiles][d] its total (workgroup = digit)
__global__ __launch_bounds__(256) void k_emb_scan(int tiles, const uint32_t* hist, uint32_t* before) {
    __shared__ uint32_t ws[4];
    const int d = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint32_t carry = 0;
    for (int b0 = 0; b0 < tiles; b0 += 256) {
        const int b = b0 + threadIdx.x;
        const uint32_t w2 = b < tiles ? hist[(int64_t)b * 128 + (d & 127)] : 0, own = d < 128 ? w2 & 0xffff : w2 >> 16;
        uint32_t v = own;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t u = __shfl_up(v, o, 64);
            if (lane >= o) v += u;
        }
        if (lane == 63) ws[w] = v;
        __syncthreads();
        uint32_t first = carry, all = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (q < w) first += ws[q];
            all += ws[q];
        }
        if (b < tiles) before[(int64_t)b * 256 + d] = first + v - own;
        carry += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) before[(int64_t)tiles * 256 + d] = carry;
}
// one pass: a tile's tokens, sorted by the digit in LDS first (so that a digit's tokens leave together),
// to their places.  7.5 us for 128 tiles: one round of latencies (keys, histograms, ranks, scans), half of it
// in the ranks' ballots and LDS counters
__global__ __launch_bounds__(RTHR) void k_emb_scatter(const void* ids, int i64, const uint2* kv, int64_t T, uint32_t V, int shift, int tiles,
                                                      const uint32_t* hist, const uint32_t* before, uint2* kv2) {
    constexpr int KPT = RTILE / RTHR;
    __shared__ RadixLds L;
    __shared__ uint32_t pre[8][256], all[8][256];
    __shared__ uint2 sh[RTILE];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t t0 = (int64_t)blockIdx.x * RTILE;
    uint32_t kk[KPT], ii[KPT], dig[KPT], rank[KPT];
    bool val[KPT];
#pragma unroll
    for (int k = 0; k < KPT; ++k) {
        const int64_t t = t0 + (w * KPT + k) * 64 + lane;
        val[k] = t < T;
        uint2 v = make_uint2(0, 0);
        if (val[k]) v = kv ? kv[t] : make_uint2(emb_key(ids, i64, t, V), (uint32_t)t);
        kk[k] = v.x;
        ii[k] = v.y;
    }
    {  // the digits' totals and their counts in earlier tiles (eight groups of threads, two digits a thread)
        const int d = threadIdx.x & 127, q = threadIdx.x >> 7;
        uint32_t p0 = 0, p1 = 0, a0 = 0, a1 = 0;
        if (before) {
            if (q == 0) {
                p0 = before[(int64_t)blockIdx.x * 256 + d];
                p1 = before[(int64_t)blockIdx.x * 256 + d + 128];
                a0 = before[(int64_t)tiles * 256 + d];
                a1 = before[(int64_t)tiles * 256 + d + 128];
            }
        } else {
            for (int b0 = q; b0 < tiles; b0 += 128) {  // 16 loads in flight
                uint32_t v[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = hist[(int64_t)min(b0 + 8 * k, tiles - 1) * 128 + d];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const int b = b0 + 8 * k;
                    const uint32_t w2 = b < tiles ? v[k] : 0, e2 = b < (int)blockIdx.x ? v[k] : 0;
                    a0 += w2 & 0xffff;
                    a1 += w2 >> 16;
                    p0 += e2 & 0xffff;
                    p1 += e2 >> 16;
                }
            }
        }
        pre[q][d] = p0;
        pre[q][d + 128] = p1;
        all[q][d] = a0;
        all[q][d + 128] = a1;
    }
#pragma unroll
    for (int k = 0; k < KPT; ++k) dig[k] = (kk[k] >> shift) & 255;
    radix_rank<KPT>(dig, val, rank, L);  // (its barriers cover pre and all)
    if (threadIdx.x < 512) {
        uint32_t(*src)[256] = threadIdx.x < 256 ? pre : all;
        const int d = threadIdx.x & 255;
        uint32_t t = 0;
#pragma unroll
        for (int q = 0; q < 8; ++q) t += src[q][d];
        if (threadIdx.x < 256) pre[0][d] = t;
        else L.tot[1][d] = t;
    }
    __syncthreads();
    digit_scan(L);  // base: the digit's first place in the tile, and of all
#pragma unroll
    for (int k = 0; k < KPT; ++k)
        if (val[k]) sh[L.base[0][dig[k]] + L.wh[w][dig[k]] + rank[k]] = make_uint2(kk[k], ii[k]);
    __syncthreads();
    const int n = T - t0 < RTILE ? (int)(T - t0) : RTILE;
    for (int j = threadIdx.x; j < n; j += RTHR) {
        const uint2 v = sh[j];
        const uint32_t d = (v.x >> shift) & 255;
        kv2[L.base[1][d] + pre[0][d] + ((uint32_t)j - L.base[0][d])] = v;
    }
}

struct EmbB {
    int64_t T;
    int N;
    int64_t Np;
    uint32_t V;
    const uint2* kv;  // the sorted tokens: id, place
    const void* ids;  // FEW: the tokens as they come
    int i64;
    const void* dy;
    int64_t lddy;
    void* out;
    float* part;      // [pieces][2][Np]: a piece's head (run from earlier pieces) and tail (run going on);
                      // FEW: [pieces][V][Np], the rows that the piece has
    uint32_t* cnt;    // FEW: [pieces][V] how many tokens
    float scale;
    int tg;           // tokens per group
};
template <class T> MMVAE_DEV void emb_out(const EmbB& a, uint32_t key, int col, const float s[8]) {
    if (key >= a.V) return;
    Chunk<T> c;
#pragma unroll
    for (int i = 0; i < 8; ++i) c.set(i, s[i] * a.scale);
    st8((T*)a.out + (int64_t)key * a.N + col, a.N - col, c);
}
static constexpr int PIECE = 1024;  // tokens of a piece at most (FEW: 512)
static constexpr uint32_t NO_KEY = 0xFFFFFFFFu;
// the piece's tokens sorted by id (V <= FEW; 256 threads, two tokens each); returns how many have a row
struct FewLds {
    uint32_t wh[4][FEW + 1], base[FEW + 1];
};
MMVAE_DEV int few_sort(const EmbB& a, int64_t p0, int P, uint32_t* sk, uint32_t* si, FewLds& L) {
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int i = threadIdx.x; i < 4 * (FEW + 1); i += 256) L.wh[i / (FEW + 1)][i % (FEW + 1)] = 0;
    __syncthreads();
    uint32_t kk[2], rank[2];
    bool val[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int j = w * 128 + k * 64 + lane;
        val[k] = j < P && p0 + j < a.T;
        kk[k] = val[k] ? emb_key(a.ids, a.i64, p0 + j, a.V) : 0;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        uint64_t m = __ballot(val[k]);
#pragma unroll
        for (int b = 0; b < 7; ++b) {
            const bool bit = (kk[k] >> b) & 1;
            const uint64_t bal = __ballot(bit);
            m &= bit ? bal : ~bal;
        }
        const uint32_t lt = __popcll(m & ((uint64_t(1) << lane) - 1));
        const uint32_t old = val[k] ? L.wh[w][kk[k]] : 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (val[k] && lt == 0) L.wh[w][kk[k]] = old + __popcll(m);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        rank[k] = old + lt;
    }
    __syncthreads();
    if (threadIdx.x < 64) {  // ids 0 .. 63: the waves' counts to offsets, then the ids'
        uint32_t t = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t c = L.wh[q][threadIdx.x];
            L.wh[q][threadIdx.x] = t;
            t += c;
        }
        const uint32_t own = t;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t u = __shfl_up(t, o, 64);
            if (lane >= o) t += u;
        }
        L.base[threadIdx.x] = t - own;
        if (threadIdx.x == 63) L.base[FEW] = t;
        if (blockIdx.y == 0 && threadIdx.x < a.V) a.cnt[(int64_t)blockIdx.x * a.V + threadIdx.x] = threadIdx.x < (uint32_t)a.V ? own : 0;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k)
        if (val[k] && kk[k] < a.V) {
            const uint32_t pos = L.base[kk[k]] + L.wh[w][kk[k]] + rank[k];
            sk[1 + pos] = kk[k];
            si[pos] = (uint32_t)(p0 + w * 128 + k * 64 + lane);
        }
    // (with V = FEW the ids outside count as FEW, with V < FEW as V: behind the rows either way)
    return (int)(a.V < FEW ? L.base[a.V] : L.base[FEW]);
}
// TPR lanes x 8 columns; the 256 / TPR groups of a workgroup take a.tg consecutive sorted tokens each, eight
// rows of dy in flight.  The groups are cut by place, not by id, so a hot id costs no more than others.
template <class T, int TPR, bool ISFEW> __global__ __launch_bounds__(256) void k_emb_seg(EmbB a) {
    constexpr int GB = 256 / TPR, U = 8;
    __shared__ float head[GB][TPR * 8], tail[GB][TPR * 8];
    __shared__ uint32_t last[GB];             // a group's last key
    __shared__ int hflag[GB], tflag[GB];      // first run goes on from before; last run goes on behind (2: one run, from before)
    __shared__ uint32_t sk[(ISFEW ? 512 : PIECE) + 2], si[ISFEW ? 512 : PIECE];  // the piece's keys, one beside each end
    const int lane = threadIdx.x % TPR, g = threadIdx.x / TPR;
    const int col = (blockIdx.y * TPR + lane) * 8;
    const int ncol = a.N - col;
    const int P = GB * a.tg;
    const int64_t p0 = (int64_t)blockIdx.x * P;
    int n;  // tokens of the piece
    if constexpr (ISFEW) {
        __shared__ FewLds L;
        n = few_sort(a, p0, P, sk, si, L);
        if (threadIdx.x == 0) {
            sk[0] = NO_KEY;
            sk[1 + n] = NO_KEY;
        }
    } else {
        n = a.T - p0 < P ? (int)(a.T - p0) : P;
        for (int i = threadIdx.x; i < n; i += 256) {
            const uint2 v = a.kv[p0 + i];
            sk[1 + i] = v.x;
            si[i] = v.y;
        }
        if (threadIdx.x == 0) {
            sk[0] = p0 > 0 ? a.kv[p0 - 1].x : NO_KEY;
            sk[1 + n] = p0 + n < a.T ? a.kv[p0 + n].x : NO_KEY;
        }
    }
    __syncthreads();
    float* part = a.part + (int64_t)blockIdx.x * (ISFEW ? (int64_t)a.V : 2) * a.Np;
    auto whole = [&](uint32_t key, const float s[8]) {  // the sum of a run that lies in the piece
        if constexpr (ISFEW) {
#pragma unroll
            for (int i = 0; i < 8; ++i) part[(int64_t)key * a.Np + col + i] = s[i];
        } else {
            emb_out<T>(a, key, col, s);
        }
    };
    const int lo = g * a.tg, hi = lo + a.tg < n ? lo + a.tg : n;
    if (lo < n) {
        uint32_t cur = sk[1 + lo];
        const bool from = sk[lo] == cur;
        bool inhead = from;  // the run being summed came from before the group
        float s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = 0.f;
        for (int t0 = lo; t0 < hi; t0 += U) {
            Chunk<T> d[U];
#pragma unroll
            for (int u = 0; u < U; ++u) d[u] = ld8((const T*)a.dy + (int64_t)si[t0 + u < hi ? t0 + u : hi - 1] * a.lddy + col, ncol);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (t0 + u >= hi) break;
                const uint32_t k = sk[1 + t0 + u];
                if (k != cur) {
                    if (inhead) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) head[g][lane * 8 + i] = s[i];
                    } else if (ncol > 0) {
                        whole(cur, s);
                    }
                    inhead = false;
                    cur = k;
#pragma unroll
                    for (int i = 0; i < 8; ++i) s[i] = 0.f;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i] += d[u].get(i);
            }
        }
        const bool on = sk[1 + hi] == cur;
        if (inhead) {
#pragma unroll
            for (int i = 0; i < 8; ++i) head[g][lane * 8 + i] = s[i];
        } else if (on) {
#pragma unroll
            for (int i = 0; i < 8; ++i) tail[g][lane * 8 + i] = s[i];
        } else if (ncol > 0) {
            whole(cur, s);
        }
        if (lane == 0) {
            last[g] = cur;
            hflag[g] = from ? 1 : 0;
            tflag[g] = on ? (inhead ? 2 : 1) : 0;
        }
    }
    __syncthreads();
    if (lo >= n || ncol <= 0) return;
    // a run over several groups is joined, in order, by the group where it begins
    const int ng = (n + a.tg - 1) / a.tg;
    float c[8];
    auto join = [&](int q) {  // adds the heads from group q on; whether the run ends in the piece
        for (; q < ng; ++q) {
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i] += head[q][lane * 8 + i];
            if (tflag[q] != 2) return true;
        }
        return false;
    };
    if (g == 0 && hflag[0]) {  // from the piece before (it may go on behind this one): the head partial
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = 0.f;
        join(0);
#pragma unroll
        for (int i = 0; i < 8; ++i) part[col + i] = c[i];
    }
    if (tflag[g] == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = tail[g][lane * 8 + i];
        if (join(g + 1)) {
            whole(last[g], c);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) part[a.Np + col + i] = c[i];
        }
    }
}
// few rows: row blockIdx.x, the pieces' partials in order (group g: pieces g, g + GB, ..)
template <class T, int TPR> __global__ __launch_bounds__(256) void k_emb_few_join(EmbB a, int pieces) {
    constexpr int GB = 256 / TPR, U = 4;
    __shared__ float sh[GB][TPR * 8];
    const int lane = threadIdx.x % TPR, g = threadIdx.x / TPR;
    const int col = (blockIdx.y * TPR + lane) * 8;
    const uint32_t v = blockIdx.x;
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = 0.f;
    if (col < a.N)
        for (int j0 = g; j0 < pieces; j0 += GB * U) {
            uint32_t has[U];
            Chunk<float> h[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = j0 + u * GB < pieces ? j0 + u * GB : j0;
                has[u] = j0 + u * GB < pieces ? a.cnt[(int64_t)j * a.V + v] : 0;
                h[u] = Chunk<float>::load(a.part + ((int64_t)j * a.V + v) * a.Np + col);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i] += has[u] ? h[u].get(i) : 0.f;  // (a row it lacks: never written)
        }
#pragma unroll
    for (int i = 0; i < 8; ++i) sh[g][lane * 8 + i] = s[i];
    __syncthreads();
    if (g != 0 || col >= a.N) return;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        for (int q = 1; q < GB; ++q) s[i] += sh[q][lane * 8 + i];
    emb_out<T>(a, v, col, s);
}
// workgroup = the run that goes on behind piece blockIdx.x and begins in it (else nothing to do)
template <class T, int TPR> __global__ __launch_bounds__(256) void k_emb_join(EmbB a, int pieces) {
    constexpr int GB = 256 / TPR;
    __shared__ float sh[GB][TPR * 8];
    __shared__ int cnt;
    const int64_t P = (int64_t)GB * a.tg;
    const int64_t c = blockIdx.x, lo = c * P, hi = lo + P;  // (hi < T: the last piece has no workgroup)
    const uint32_t key = a.kv[hi].x;
    if (key >= a.V || a.kv[hi - 1].x != key) return;
    if (c > 0 && a.kv[lo - 1].x == key) return;  // begins in an earlier piece (the keys are sorted)
    if (threadIdx.x == 0) cnt = 0;
    __syncthreads();
    // pieces behind c that the run fills to their end and beyond
    for (int64_t j0 = c + 1; j0 < pieces; j0 += 256) {
        const int64_t j = j0 + threadIdx.x, e = (j + 1) * P;
        const bool in = j < pieces && e < a.T && a.kv[e].x == key;
        const uint64_t m = __ballot(in);
        if ((threadIdx.x & 63) == 0 && m) atomicAdd(&cnt, __popcll(m));
        const int64_t e1 = (j0 + 256) * P;  // the last of these pieces
        if (e1 >= a.T || a.kv[e1].x != key) break;
    }
    __syncthreads();
    const int64_t end = c + 1 + cnt;  // the last piece of the run
    const int lane = threadIdx.x % TPR, g = threadIdx.x / TPR;
    const int col = (blockIdx.y * TPR + lane) * 8;
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = 0.f;
    if (col < a.N)
        for (int64_t j0 = c + 1 + g; j0 <= end; j0 += GB * 4) {
            Chunk<float> h[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) h[u] = Chunk<float>::load(a.part + (j0 + u * GB <= end ? j0 + u * GB : j0) * 2 * a.Np + col);
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i] += j0 + u * GB <= end ? h[u].get(i) : 0.f;
        }
#pragma unroll
    for (int i = 0; i < 8; ++i) sh[g][lane * 8 + i] = s[i];
    __syncthreads();
    if (g != 0 || col >= a.N) return;
    const Chunk<float> t = Chunk<float>::load(a.part + c * 2 * a.Np + a.Np + col);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        s[i] = t.get(i);
        for (int q = 0; q < GB; ++q) s[i] += sh[q][lane * 8 + i];
    }
    emb_out<T>(a, key, col, s);
}

// =======================================================================================
// Host side
// =======================================================================================
hipError_t norm_fwd(const mmvae_norm_args& a, hipStream_t st) {
    if (a.M == 0) return hipSuccess;
    return a.dtype == MMVAE_T_F32 ? norm_fwd_f32(a, st) : a.dtype == MMVAE_T_BF16 ? norm_fwd_bf16(a, st) : norm_fwd_f16(a, st);
}
hipError_t norm_bwd(const mmvae_norm_args& a, hipStream_t st) {
    return a.dtype == MMVAE_T_F32 ? norm_bwd_f32(a, st) : a.dtype == MMVAE_T_BF16 ? norm_bwd_bf16(a, st) : norm_bwd_f16(a, st);
}

hipError_t dropout(const mmvae_dropout_args& a, hipStream_t st) {
    if (a.M == 0 || a.N == 0) return hipSuccess;
    const DropKey k = drop_key(a.p, a.seed, a.step, a.row_offset, a.state);
    return by_type(a.dtype, [&](auto ty) -> hipError_t {
        using T = decltype(ty);
        return launch(k_dropout<T>, dim3((unsigned)walk_blocks(a.M, a.N)), dim3(256), st, a.M, (int)a.N, (const T*)a.x, a.ldx, (T*)a.y, a.ldy, k);
    });
}

hipError_t emb_fwd(const mmvae_embedding_args& a, hipStream_t st) {
    if (a.T == 0) return hipSuccess;
    EmbF p;
    p.T = a.T;
    p.N = (int)a.N;
    p.V = a.V;
    p.ids = a.ids;
    p.table = a.table;
    p.add = a.add;
    p.ldt = a.ldt;
    p.ldadd = a.ldadd;
    p.ldy = a.ldy;
    p.y = a.y;
    p.scale = a.scale;
    p.i64 = a.ids64;
    return by_type(a.dtype, [&](auto ty) -> hipError_t {
        return launch(k_emb_fwd<decltype(ty)>, dim3((unsigned)walk_blocks(a.T, a.N)), dim3(256), st, p);
    });
}

// the gradient's plan, a function of (T, N, V) alone: tokens per group and pieces
static constexpr int64_t SHORT_T = 32768;  // up to so many tokens a group takes 8
struct EmbPlan {
    bool few;
    int tpr, gb, tg, slices;
    int64_t pieces, tiles, Np;
    int64_t o_kv[2], o_hist, o_before, o_part, bytes;
};
static EmbPlan emb_plan(int64_t T, int64_t N, int64_t V) {
    EmbPlan q;
    std::memset(&q, 0, sizeof(q));
    const int64_t nc = (N + 7) / 8;
    q.Np = nc * 8;
    q.few = V <= FEW;
    // lanes a row: 32, or 16 where 32 would leave over a fifth more of them idle (262144 x 128 bf16: 16 lanes
    // 15.6 us, 32 23.1 us; 50001 x 517 f16: 16 lanes 25.1 us, 32 23.3 us, 64 22.9 us, 8 29.6 us)
    auto lanes = [&](int64_t t) { return (nc + t - 1) / t * t; };
    q.tpr = nc <= 8 ? 8 : 5 * lanes(32) > 6 * lanes(16) ? 16 : 32;
    q.gb = 256 / q.tpr;
    q.slices = (int)((nc + q.tpr - 1) / q.tpr);
    // a group's tokens: 8 in one go of loads; more for long inputs, so that the partials stay few beside dy
    q.tg = T > SHORT_T ? 16 : 8;
    if (q.few && T > SHORT_T) q.tg = 512 / q.gb;
    q.pieces = std::max<int64_t>(1, (T + (int64_t)q.gb * q.tg - 1) / ((int64_t)q.gb * q.tg));
    q.tiles = (T + RTILE - 1) / RTILE;
    int64_t o = 0;
    auto take = [&](int64_t b) {
        const int64_t at = o;
        o += (b + 255) / 256 * 256;
        return at;
    };
    if (!q.few)
        for (int i = 0; i < (T <= RONE ? 1 : 2); ++i) q.o_kv[i] = take(T * 8);
    q.o_hist = take(q.few ? q.pieces * V * 4 : q.tiles * 128 * 4);
    q.o_before = take(!q.few && q.tiles > RFUSE ? (q.tiles + 1) * 256 * 4 : 0);
    q.o_part = take(q.pieces * (q.few ? V : 2) * q.Np * 4);
    q.bytes = o;
    return q;
}
static int64_t emb_need(int64_t T, int64_t N, int64_t V) { return T == 0 || V == 0 ? 0 : emb_plan(T, N, V).bytes; }
// enough for T tokens and for any fewer: on each side of SHORT_T the need grows with T, but above it a group takes
// more tokens, so that there are fewer partials (12 rows of 128: 32768 tokens 1.6 MB, 32769 0.4 MB)
int64_t emb_bwd_ws(int64_t T, int64_t N, int64_t V) { return std::max(emb_need(T, N, V), emb_need(std::min(T, SHORT_T), N, V)); }

__global__ __launch_bounds__(1024) void k_emb_clear(void* out, int64_t out_bytes) {
    fill_zero(out, out_bytes, (int64_t)blockIdx.x * 1024 + threadIdx.x, (int64_t)gridDim.x * 1024);
}

hipError_t emb_bwd(const mmvae_embedding_args& a, hipStream_t st) {
    const int64_t z = a.dtype == MMVAE_T_F32 ? 4 : 2, out_bytes = a.V * a.N * z;
    const int clear = (int)std::min<int64_t>((out_bytes / 4 + RTHR * 4 - 1) / (RTHR * 4) + 1, 1024);
    if (out_bytes == 0) return hipSuccess;
    if (a.T == 0) return launch(k_emb_clear, dim3((unsigned)clear), dim3(1024), st, a.dtable, out_bytes);
    const EmbPlan q = emb_plan(a.T, a.N, a.V);
    char* ws = (char*)a.ws;
    uint2* kv[2] = {(uint2*)(ws + q.o_kv[0]), (uint2*)(ws + q.o_kv[1])};
    uint32_t* hist = (uint32_t*)(ws + q.o_hist);
    const uint32_t V = (uint32_t)a.V;
    int passes = 1;
    while (passes < 4 && (V >> (8 * passes)) != 0) ++passes;
    int cur = 0;
    if (!q.few && a.T <= RONE) {
        OPCHK(launch(k_emb_sort1, dim3((unsigned)(1 + clear)), dim3(RTHR), st, a.ids, a.ids64, (int)a.T, V, passes, kv[0], a.dtable, out_bytes));
    } else if (!q.few) {
        const int tiles = (int)q.tiles;
        uint32_t* before = tiles > RFUSE ? (uint32_t*)(ws + q.o_before) : nullptr;
        for (int p = 0; p < passes; ++p) {
            const uint2* from = p ? kv[cur] : nullptr;
            const int nxt = p ? cur ^ 1 : 0;
            OPCHK(launch(k_emb_hist, dim3((unsigned)(tiles + (p ? 0 : clear))), dim3(RTHR), st, a.ids, a.ids64, from, a.T, V, 8 * p, tiles,
                         hist, a.dtable, out_bytes));
            if (before) OPCHK(launch(k_emb_scan, dim3(256), dim3(256), st, tiles, (const uint32_t*)hist, before));
            OPCHK(launch(k_emb_scatter, dim3((unsigned)tiles), dim3(RTHR), st, a.ids, a.ids64, from, a.T, V, 8 * p, tiles,
                         (const uint32_t*)hist, (const uint32_t*)before, kv[nxt]));
            cur = nxt;
        }
    }
    EmbB b;
    std::memset(&b, 0, sizeof(b));
    b.T = a.T;
    b.N = (int)a.N;
    b.Np = q.Np;
    b.V = V;
    b.kv = kv[cur];
    b.ids = a.ids;
    b.i64 = a.ids64;
    b.dy = a.dy;
    b.lddy = a.lddy;
    b.out = a.dtable;
    b.part = (float*)(ws + q.o_part);
    b.cnt = hist;
    b.scale = a.scale;
    b.tg = q.tg;
    const dim3 grid((unsigned)q.pieces, (unsigned)q.slices), jgrid((unsigned)(q.pieces - 1), (unsigned)q.slices);
    const dim3 fgrid((unsigned)a.V, (unsigned)q.slices);
    return by_type(a.dtype, [&](auto ty) -> hipError_t {
        using T = decltype(ty);
        auto go = [&](auto t) -> hipError_t {
            if (q.few) {
                OPCHK(launch(k_emb_seg<T, t.value, true>, grid, dim3(256), st, b));
                return launch(k_emb_few_join<T, t.value>, fgrid, dim3(256), st, b, (int)q.pieces);
            }
            OPCHK(launch(k_emb_seg<T, t.value, false>, grid, dim3(256), st, b));
            return q.pieces > 1 ? launch(k_emb_join<T, t.value>, jgrid, dim3(256), st, b, (int)q.pieces) : hipSuccess;
        };
        if (q.tpr == 8) return go(I<8>{});
        if (q.tpr == 16) return go(I<16>{});
        return go(I<32>{});
    });
}

// ---- argument checks: null, or what is wrong -------------------------------------------------
static bool type_ok(int t) { return t == MMVAE_T_F32 || t == MMVAE_T_BF16 || t == MMVAE_T_F16; }
static constexpr int64_t MAX_DIM = (int64_t(1) << 31) - 65536;  // rows, widths, tokens and table rows
static constexpr int64_t MAX_WALK = (int64_t(1) << 24) - 1;     // workgroups of 256 threads: a grid has below 2^32 threads
static bool aligned(const void* p, int type) { return ((uintptr_t)p & (type == MMVAE_T_F32 ? 3 : 1)) == 0; }
static bool ld_ok(int64_t ld, int64_t N, int64_t M) { return M <= 1 || ld >= N; }  // an output's rows may not overlap
static const char* drop_check(double p) { return p >= 0. && p <= 1. ? nullptr : "p must be in [0, 1]"; }

const char* norm_check(const mmvae_norm_args& a, bool bwd) {
    if (a.M < 0 || a.N < 1 || a.M > MAX_DIM || a.N > MAX_DIM) return "need 0 <= M < 2^31 rows and 1 <= N < 2^31 columns";
    if (!type_ok(a.dtype) || (a.wtype != a.dtype && a.wtype != MMVAE_T_F32))
        return "types: f32, bf16 or f16; weight and bias of the same type or f32";
    if (!(a.eps >= 0.f) || std::isinf(a.eps)) return "eps must be finite and >= 0";
    if (const char* m = drop_check(a.p)) return m;
    if (a.ldx < 0 || a.lddy < 0) return "row strides must be >= 0";
    if (a.M > 0 && !a.x) return "x is null";
    for (const void* p : {a.x, (const void*)a.y, a.dy, (const void*)a.dx})
        if (!aligned(p, a.dtype)) return "x, y, dy and dx must be aligned to their type";
    for (const void* p : {a.w, a.b, (const void*)a.dw, (const void*)a.db})
        if (!aligned(p, a.wtype)) return "w, b, dw and db must be aligned to their type";
    for (const void* p : {(const void*)a.mean, (const void*)a.rstd, (const void*)a.ws})
        if (!aligned(p, MMVAE_T_F32)) return "mean, rstd and the workspace must be 4-byte aligned";
    if (((uintptr_t)a.state & 7) != 0) return "state must be 8-byte aligned";
    if (!bwd) {
        if (a.M > 0 && !a.y) return "y is null";
        if (!ld_ok(a.ldy, a.N, a.M)) return "y's row stride is below N";
        return nullptr;
    }
    if (a.M > 0 && (!a.dy || !a.mean || !a.rstd)) return "dy, mean or rstd is null";
    if (a.dx && !ld_ok(a.lddx, a.N, a.M)) return "dx's row stride is below N";
    // (k_ln_wred: 1024 threads for 32 of the 2 x padded width's sums, and a grid has below 2^32 threads)
    if ((a.dw || a.db) && a.N > (1 << 26) - 16) return "need N <= 2^26 - 16 with dw or db";
    if ((a.dw || a.db) && norm_bwd_ws(a.M, a.N) > 0 && (!a.ws || a.ws_bytes < norm_bwd_ws(a.M, a.N)))
        return "the workspace is below mmvae_layer_norm_bwd_ws(M, N) bytes";
    return nullptr;
}
const char* dropout_check(const mmvae_dropout_args& a) {
    if (a.M < 0 || a.N < 0 || a.M > MAX_DIM || a.N > MAX_DIM) return "need 0 <= M, N < 2^31";
    if (a.M > 0 && a.N > 0 && (a.N >= (1 << 24) || walk_blocks(a.M, a.N) > MAX_WALK)) return "need N < 2^24, and M N below 2^37";
    if (!type_ok(a.dtype)) return "types: f32, bf16 or f16";
    if (!aligned(a.x, a.dtype) || !aligned(a.y, a.dtype) || ((uintptr_t)a.state & 7) != 0) return "x, y and state must be aligned to their types";
    if (const char* m = drop_check(a.p)) return m;
    if (a.M > 0 && a.N > 0 && (!a.x || !a.y)) return "x or y is null";
    if (a.ldx < 0 || !ld_ok(a.ldy, a.N, a.M)) return "x's row stride is negative or y's below N";
    return nullptr;
}
const char* emb_check(const mmvae_embedding_args& a, bool bwd) {
    if (a.T < 0 || a.N < 1 || a.V < 0 || a.T > MAX_DIM || a.N >= (1 << 24) || a.V > MAX_DIM)
        return "need 0 <= T, V < 2^31 and 1 <= N < 2^24";
    if (!type_ok(a.dtype)) return "types: f32, bf16 or f16";
    if (walk_blocks(a.T, a.N) > MAX_WALK) return "need T N below 2^37";
    for (const void* p : {a.table, a.add, (const void*)a.y, a.dy})
        if (!aligned(p, a.dtype)) return "table, add, y and dy must be aligned to their type";
    if (((uintptr_t)a.ids & (a.ids64 ? 7 : 3)) != 0) return "ids must be aligned to their type";
    if (a.T > 0 && !a.ids) return "ids is null";
    if (!bwd) {
        if (a.T > 0 && a.V > 0 && !a.table) return "table is null";
        if (a.T > 0 && !a.y) return "y is null";
        if (a.ldt < 0 || a.ldadd < 0 || !ld_ok(a.ldy, a.N, a.T)) return "a row stride is negative, or y's below N";
        return nullptr;
    }
    if (a.T > 0 && !a.dy) return "dy is null";
    if (a.V > 0 && !a.dtable) return "dtable is null";
    if (a.lddy < 0) return "dy's row stride is negative";
    if ((uintptr_t)a.dtable & 3) return "dtable must be 4-byte aligned";
    if (emb_need(a.T, a.N, a.V) > 0 && (!a.ws || a.ws_bytes < emb_need(a.T, a.N, a.V)))
        return "the workspace is below mmvae_embedding_bwd_ws(T, N, V) bytes";
    if (((uintptr_t)a.ws & 15) != 0) return "the workspace must be 16-byte aligned";
    return nullptr;
}

}  // namespace mmvae

using namespace mmvae;

// the caller's device for the length of a call
struct OnDevice {
    int before = -1;
    hipError_t er;
    explicit OnDevice(int d) {
        er = hipGetDevice(&before);
        if (er == hipSuccess && before != d) er = hipSetDevice(d);
        else before = -1;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};
template <class A, class F> static int op_call(const char* name, const A* a, const char* wrong, F&& f) {
    if (wrong) return set_last_error(MMVAE_E_ARG, name, wrong);
    OnDevice on(a->device);
    const hipError_t er = on.er == hipSuccess ? f(*a, (hipStream_t)a->stream) : on.er;
    if (er == hipSuccess) return MMVAE_OK;
    return set_last_error(MMVAE_E_HIP, name, hipGetErrorString(er));
}

extern "C" {

int mmvae_layer_norm_fwd(const mmvae_norm_args* a) {
    return op_call("layer_norm_fwd", a, a ? norm_check(*a, false) : "null arguments", norm_fwd);
}
int mmvae_layer_norm_bwd(const mmvae_norm_args* a) {
    return op_call("layer_norm_bwd", a, a ? norm_check(*a, true) : "null arguments", norm_bwd);
}
int64_t mmvae_layer_norm_bwd_ws(int64_t M, int64_t N) { return M < 0 || N < 1 ? 0 : norm_bwd_ws(M, N); }
int mmvae_dropout(const mmvae_dropout_args* a) {
    return op_call("dropout", a, a ? dropout_check(*a) : "null arguments", dropout);
}
int mmvae_embedding_fwd(const mmvae_embedding_args* a) {
    return op_call("embedding_fwd", a, a ? emb_check(*a, false) : "null arguments", emb_fwd);
}
int mmvae_embedding_bwd(const mmvae_embedding_args* a) {
    return op_call("embedding_bwd", a, a ? emb_check(*a, true) : "null arguments", emb_bwd);
}
int64_t mmvae_embedding_bwd_ws(int64_t T, int64_t N, int64_t V) { return T < 0 || N < 1 || V < 0 ? 0 : emb_bwd_ws(T, N, V); }

}  // extern "C"
