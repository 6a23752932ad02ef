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
// Dropout alone: tpr = 2^s threads walk a row's chunks, 256 / tpr rows per workgroup
// =======================================================================================
template <class T>
__global__ __launch_bounds__(256) void k_dropout(int64_t M, int64_t N, const T* x, int64_t ldx, T* y, int64_t ldy, int ltpr, DropKey k) {
    const int tpr = 1 << ltpr, rpb = 256 >> ltpr;
    const int lane = threadIdx.x & (tpr - 1), grp = threadIdx.x >> ltpr;
    drop_state(k);
    for (int64_t row = (int64_t)blockIdx.x * rpb + grp; row < M; row += (int64_t)gridDim.x * rpb) {
        const T* xr = x + row * ldx;
        T* yr = y + row * ldy;
        for (int64_t col = lane * 8; col < N; col += tpr * 8) {
            const int n = (int)(N - col < 8 ? N - col : 8);
            Chunk<T> c = ld8(xr + col, n);
            bool kept[8];
            keep8(k, row, (int)(col >> 3), kept);
#pragma unroll
            for (int i = 0; i < 8; ++i) c.set(i, kept[i] ? c.get(i) * k.s : 0.f);
            st8(yr + col, n, c);
        }
    }
}

// =======================================================================================
// Embedding: y[t] = scale table[id_t] (+ add[t]), zero rows for ids outside [0, V)
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
template <class T> __global__ __launch_bounds__(256) void k_emb_fwd(EmbF a, int ltpr) {
    const int tpr = 1 << ltpr, rpb = 256 >> ltpr;
    const int lane = threadIdx.x & (tpr - 1), grp = threadIdx.x >> ltpr;
    for (int64_t t = (int64_t)blockIdx.x * rpb + grp; t < a.T; t += (int64_t)gridDim.x * rpb) {
        const int64_t id = emb_id(a.ids, a.i64, t);
        const bool ok = id >= 0 && id < a.V;
        const T* tr = (const T*)a.table + (ok ? id : 0) * a.ldt;
        T* yr = (T*)a.y + t * a.ldy;
        for (int col = lane * 8; col < a.N; col += tpr * 8) {
            const int n = a.N - col;
            Chunk<T> c = ld8(tr + col, ok ? n : 0);
            if (a.add) {
                const Chunk<T> d = ld8((const T*)a.add + t * a.ldadd + col, n);
#pragma unroll
                for (int i = 0; i < 8; ++i) c.set(i, ok ? __builtin_fmaf(c.get(i), a.scale, d.get(i)) : d.get(i));
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) c.set(i, ok ? c.get(i) * a.scale : 0.f);
            }
            st8(yr + col, n, c);
        }
    }
}

// =======================================================================================
// Embedding gradient: dE[v] = scale sum over the tokens of v of dy.
//   1. the tokens sorted by id, stable (LSD radix sort, 8-bit digits; ids outside [0, V) as V,
//      behind all others): in one workgroup up to 4096 tokens, else histogram + scatter per digit;
//   2. k_emb_seg: fixed pieces of the sorted tokens, whatever their ids: a hot id is spread over
//      many workgroups, the sums of runs inside a piece are final, the first and last run of a
//      piece leave a partial where they go on in the next one;
//   3. k_emb_join: the partials of a run that crosses pieces, summed in order.
// =======================================================================================
static constexpr int RTILE = 4096, RTHR = 1024, RKPT = RTILE / RTHR;  // a sort tile: 16 waves x 4 x 64 tokens
static constexpr int RFUSE = 128;  // up to so many tiles a scatter workgroup sums the histograms itself

// stable ranks of the workgroup's keys by an 8-bit digit (16 waves, RKPT keys a lane; wave w holds the
// tokens w 256 + k 64 + lane).  wh[w][d]: first the wave's counts, then the count of d in earlier waves.
struct RadixLds {
    uint32_t wh[RTHR / 64][256];
    uint32_t tot[256];   // the tile's count of each digit
    uint32_t base[256];  // exclusive sums of tot
    uint32_t ws[4];
};
MMVAE_DEV void radix_rank(const uint32_t dig[RKPT], const bool val[RKPT], uint32_t rank[RKPT], RadixLds& L) {
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int i = threadIdx.x; i < (RTHR / 64) * 256; i += RTHR) L.wh[i >> 8][i & 255] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < RKPT; ++k) {
        uint64_t m = __ballot(val[k]);
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const bool bit = (dig[k] >> b) & 1;
            const uint64_t bal = __ballot(bit);
            m &= bit ? bal : ~bal;
        }
        const uint32_t lt = __popcll(m & ((uint64_t(1) << lane) - 1));
        const uint32_t old = val[k] ? L.wh[w][dig[k]] : 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (val[k] && lt == 0) L.wh[w][dig[k]] = old + __popcll(m);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        rank[k] = old + lt;
    }
    __syncthreads();
    uint32_t t = 0;
    if (threadIdx.x < 256) {
#pragma unroll
        for (int q = 0; q < RTHR / 64; ++q) {
            const uint32_t c = L.wh[q][threadIdx.x];
            L.wh[q][threadIdx.x] = t;
            t += c;
        }
        L.tot[threadIdx.x] = t;
    }
    __syncthreads();
}
// base[d] = sum of src[e] over e < d (256 digits, waves 0 .. 3)
MMVAE_DEV void digit_scan(const uint32_t* src, RadixLds& L) {
    uint32_t own = 0, v = 0;
    if (threadIdx.x < 256) {
        own = v = src[threadIdx.x];
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t u = __shfl_up(v, o, 64);
            if ((int)(threadIdx.x & 63) >= o) v += u;
        }
        if ((threadIdx.x & 63) == 63) L.ws[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    if (threadIdx.x < 256) {
        uint32_t b = v - own;
        for (int q = 0; q < (int)(threadIdx.x >> 6); ++q) b += L.ws[q];
        L.base[threadIdx.x] = b;
    }
    __syncthreads();
}
MMVAE_DEV uint32_t emb_key(const void* ids, int i64, int64_t t, uint32_t V) {
    const int64_t id = emb_id(ids, i64, t);
    return id >= 0 && id < (int64_t)V ? (uint32_t)id : V;
}
MMVAE_DEV void fill_zero(uint32_t* out, int64_t words, int64_t i, int64_t step) {  // out 4-byte aligned
    for (; i < words; i += step) out[i] = 0;
}

// the whole sort of T <= RTILE tokens in workgroup 0; the others clear the gradient
__global__ __launch_bounds__(RTHR) void k_emb_sort1(const void* ids, int i64, int T, uint32_t V, int passes, uint32_t* key,
                                                    uint32_t* idx, void* out, int64_t out_bytes) {
    if (blockIdx.x > 0) {
        fill_zero((uint32_t*)out, out_bytes / 4, (int64_t)(blockIdx.x - 1) * RTHR + threadIdx.x, (int64_t)(gridDim.x - 1) * RTHR);
        if (blockIdx.x == 1 && threadIdx.x == 0 && (out_bytes & 2)) ((uint16_t*)out)[out_bytes / 2 - 1] = 0;
        return;
    }
    __shared__ RadixLds L;
    __shared__ uint32_t sk[RTILE], si[RTILE];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    uint32_t kk[RKPT], ii[RKPT], dig[RKPT], rank[RKPT];
    bool val[RKPT];
#pragma unroll
    for (int k = 0; k < RKPT; ++k) {
        const int t = w * 256 + k * 64 + lane;
        val[k] = t < T;
        kk[k] = val[k] ? emb_key(ids, i64, t, V) : 0;
        ii[k] = t;
    }
    for (int p = 0; p < passes; ++p) {
#pragma unroll
        for (int k = 0; k < RKPT; ++k) dig[k] = (kk[k] >> (8 * p)) & 255;
        radix_rank(dig, val, rank, L);
        digit_scan(L.tot, L);
#pragma unroll
        for (int k = 0; k < RKPT; ++k)
            if (val[k]) {
                const uint32_t pos = L.base[dig[k]] + L.wh[w][dig[k]] + rank[k];
                sk[pos] = kk[k];
                si[pos] = ii[k];
            }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < RKPT; ++k) {
            const int t = w * 256 + k * 64 + lane;
            if (t < T) {
                kk[k] = sk[t];
                ii[k] = si[t];
            }
        }
    }
#pragma unroll
    for (int k = 0; k < RKPT; ++k) {
        const int t = w * 256 + k * 64 + lane;
        if (t < T) {
            key[t] = kk[k];
            idx[t] = ii[k];
        }
    }
}

// digit counts of each tile: hist[tile][256]; key null: the first pass, from the ids.  Workgroups past
// the tiles (first pass) clear the gradient.
__global__ __launch_bounds__(RTHR) void k_emb_hist(const void* ids, int i64, const uint32_t* key, int64_t T, uint32_t V, int shift,
                                                   int tiles, uint32_t* hist, void* out, int64_t out_bytes) {
    if ((int)blockIdx.x >= tiles) {
        const int b = blockIdx.x - tiles, nb = gridDim.x - tiles;
        fill_zero((uint32_t*)out, out_bytes / 4, (int64_t)b * RTHR + threadIdx.x, (int64_t)nb * RTHR);
        if (b == 0 && threadIdx.x == 0 && (out_bytes & 2)) ((uint16_t*)out)[out_bytes / 2 - 1] = 0;
        return;
    }
    __shared__ uint32_t h[256];
    if (threadIdx.x < 256) h[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < RKPT; ++k) {
        const int64_t t = (int64_t)blockIdx.x * RTILE + k * RTHR + threadIdx.x;
        if (t < T) atomicAdd(&h[((key ? key[t] : emb_key(ids, i64, t, V)) >> shift) & 255], 1u);
    }
    __syncthreads();
    if (threadIdx.x < 256) hist[(int64_t)blockIdx.x * 256 + threadIdx.x] = h[threadIdx.x];
}
// many tiles: hist[.][d] -> the count of d in earlier tiles, hist[tiles][d] its total (workgroup = digit)
__global__ __launch_bounds__(256) void k_emb_scan(int tiles, uint32_t* hist) {
    __shared__ uint32_t ws[4];
    const int d = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint32_t carry = 0;
    for (int b0 = 0; b0 < tiles; b0 += 256) {
        const int b = b0 + threadIdx.x;
        const uint32_t own = b < tiles ? hist[(int64_t)b * 256 + d] : 0;
        uint32_t v = own;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t u = __shfl_up(v, o, 64);
            if (lane >= o) v += u;
        }
        if (lane == 63) ws[w] = v;
        __syncthreads();
        uint32_t before = carry, all = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (q < w) before += ws[q];
            all += ws[q];
        }
        if (b < tiles) hist[(int64_t)b * 256 + d] = before + v - own;
        carry += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) hist[(int64_t)tiles * 256 + d] = carry;
}
__global__ __launch_bounds__(RTHR) void k_emb_scatter(const void* ids, int i64, const uint32_t* key, const uint32_t* idx, int64_t T,
                                                      uint32_t V, int shift, int tiles, int scanned, const uint32_t* hist,
                                                      uint32_t* key2, uint32_t* idx2) {
    __shared__ RadixLds L;
    __shared__ uint32_t pre[4][256], all[4][256];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    {  // the digits' totals and their counts in earlier tiles
        const int d = threadIdx.x & 255, q = threadIdx.x >> 8;
        uint32_t p = 0, t = 0;
        if (scanned) {
            if (q == 0) {
                p = hist[(int64_t)blockIdx.x * 256 + d];
                t = hist[(int64_t)tiles * 256 + d];
            }
        } else {
            for (int b = q; b < tiles; b += 4) {
                const uint32_t v = hist[(int64_t)b * 256 + d];
                t += v;
                if (b < (int)blockIdx.x) p += v;
            }
        }
        pre[q][d] = p;
        all[q][d] = t;
    }
    __syncthreads();
    if (threadIdx.x < 256) {
        const int d = threadIdx.x;
        pre[0][d] = pre[0][d] + pre[1][d] + pre[2][d] + pre[3][d];
        all[0][d] = all[0][d] + all[1][d] + all[2][d] + all[3][d];
    }
    __syncthreads();
    digit_scan(all[0], L);
    uint32_t kk[RKPT], ii[RKPT], dig[RKPT], rank[RKPT];
    bool val[RKPT];
#pragma unroll
    for (int k = 0; k < RKPT; ++k) {
        const int64_t t = (int64_t)blockIdx.x * RTILE + w * 256 + k * 64 + lane;
        val[k] = t < T;
        kk[k] = val[k] ? (key ? key[t] : emb_key(ids, i64, t, V)) : 0;
        ii[k] = val[k] && idx ? idx[t] : (uint32_t)t;
        dig[k] = (kk[k] >> shift) & 255;
    }
    radix_rank(dig, val, rank, L);
#pragma unroll
    for (int k = 0; k < RKPT; ++k)
        if (val[k]) {
            const uint32_t pos = L.base[dig[k]] + pre[0][dig[k]] + L.wh[w][dig[k]] + rank[k];
            key2[pos] = kk[k];
            idx2[pos] = ii[k];
        }
}

struct EmbB {
    int64_t T;
    int N;
    int64_t Np;
    uint32_t V;
    const uint32_t *key, *idx;
    const void* dy;
    int64_t lddy;
    void* out;
    float* part;  // [pieces][2][Np]: a piece's head (run from earlier pieces) and tail (run going on)
    float scale;
    int tg;       // tokens per group
};
template <class T> MMVAE_DEV void emb_out(const EmbB& a, uint32_t key, int col, const float s[8]) {
    if (key >= a.V) return;
    Chunk<T> c;
#pragma unroll
    for (int i = 0; i < 8; ++i) c.set(i, s[i] * a.scale);
    st8((T*)a.out + (int64_t)key * a.N + col, a.N - col, c);
}
// TPR lanes x 8 columns; the 256 / TPR groups of a workgroup take a.tg consecutive sorted tokens each
template <class T, int TPR> __global__ __launch_bounds__(256) void k_emb_seg(EmbB a) {
    constexpr int GB = 256 / TPR, U = 8;
    __shared__ float head[GB][TPR * 8], tail[GB][TPR * 8];
    __shared__ uint32_t first[GB], last[GB];  // a group's first and last key
    __shared__ int hflag[GB], tflag[GB];      // first run goes on from before; last run goes on behind (2: one run, from before)
    const int lane = threadIdx.x % TPR, g = threadIdx.x / TPR;
    const int col = (blockIdx.y * TPR + lane) * 8;
    const int ncol = a.N - col;
    const int64_t p0 = (int64_t)blockIdx.x * GB * a.tg;
    const int64_t lo = p0 + (int64_t)g * a.tg, hi = lo + a.tg < a.T ? lo + a.tg : a.T;
    const bool any = lo < a.T;
    if (any) {
        uint32_t cur = a.key[lo];
        const bool from = lo > 0 && a.key[lo - 1] == cur;
        bool inhead = from;  // the run being summed came from before the group
        float s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = 0.f;
        for (int64_t t0 = lo; t0 < hi; t0 += U) {
            uint32_t kk[U];
            Chunk<T> d[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t t = t0 + u < hi ? t0 + u : hi - 1;
                kk[u] = a.key[t];
                d[u] = ld8((const T*)a.dy + (int64_t)a.idx[t] * a.lddy + col, ncol);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (t0 + u >= hi) break;
                if (kk[u] != cur) {
                    if (inhead) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) head[g][lane * 8 + i] = s[i];
                    } else if (ncol > 0) {
                        emb_out<T>(a, cur, col, s);
                    }
                    inhead = false;
                    cur = kk[u];
#pragma unroll
                    for (int i = 0; i < 8; ++i) s[i] = 0.f;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i] += d[u].get(i);
            }
        }
        const bool on = hi < a.T && a.key[hi] == cur;
        if (inhead) {
#pragma unroll
            for (int i = 0; i < 8; ++i) head[g][lane * 8 + i] = s[i];
        } else if (on) {
#pragma unroll
            for (int i = 0; i < 8; ++i) tail[g][lane * 8 + i] = s[i];
        } else if (ncol > 0) {
            emb_out<T>(a, cur, col, s);
        }
        if (lane == 0) {
            first[g] = a.key[lo];
            last[g] = cur;
            hflag[g] = from ? 1 : 0;
            tflag[g] = on ? (inhead ? 2 : 1) : 0;
        }
    }
    __syncthreads();
    if (g != 0 || ncol <= 0) return;
    // the groups' open runs joined in order by the first group's lanes
    float c[8];
    bool open = false, prev = false;
    uint32_t ck = 0;
    float* part = a.part + (int64_t)blockIdx.x * 2 * a.Np;
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = 0.f;
    for (int q = 0; q < GB && p0 + (int64_t)q * a.tg < a.T; ++q) {
        if (hflag[q]) {
            if (q == 0) {
                prev = true;
#pragma unroll
                for (int i = 0; i < 8; ++i) c[i] = head[0][lane * 8 + i];
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) c[i] += head[q][lane * 8 + i];
            }
            open = true;
            ck = first[q];
            if (tflag[q] == 2) continue;  // the whole group is inside the run
            if (prev) {
#pragma unroll
                for (int i = 0; i < 8; ++i) part[col + i] = c[i];
            } else {
                emb_out<T>(a, ck, col, c);
            }
            open = prev = false;
        }
        if (tflag[q] == 1) {
            open = true;
            prev = false;
            ck = last[q];
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i] = tail[q][lane * 8 + i];
        }
    }
    if (open) {  // goes on in the next piece
        float* o = part + (prev ? 0 : a.Np);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[col + i] = c[i];
    }
}
// workgroup = the run that goes on behind piece blockIdx.x and begins in it (else nothing to do)
template <class T, int TPR> __global__ __launch_bounds__(256) void k_emb_join(EmbB a, int pieces) {
    constexpr int GB = 256 / TPR;
    __shared__ float sh[GB][TPR * 8];
    __shared__ int cnt;
    const int64_t P = (int64_t)GB * a.tg;
    const int64_t c = blockIdx.x, lo = c * P, hi = lo + P;  // (hi < T: the last piece has no workgroup)
    const uint32_t key = a.key[hi];
    if (key >= a.V || a.key[hi - 1] != key) return;
    if (c > 0 && a.key[lo - 1] == key) return;  // begins in an earlier piece (the keys are sorted)
    if (threadIdx.x == 0) cnt = 0;
    __syncthreads();
    // pieces behind c that the run fills to their end and beyond
    for (int64_t j0 = c + 1; j0 < pieces; j0 += 256) {
        const int64_t j = j0 + threadIdx.x, e = (j + 1) * P;
        const bool in = j < pieces && e < a.T && a.key[e] == key;
        const uint64_t m = __ballot(in);
        if ((threadIdx.x & 63) == 0 && m) atomicAdd(&cnt, __popcll(m));
        const int64_t e1 = (j0 + 256) * P;  // the last of these pieces
        if (e1 >= a.T || a.key[e1] != key) break;
    }
    __syncthreads();
    const int64_t end = c + 1 + cnt;  // the last piece of the run
    const int lane = threadIdx.x % TPR, g = threadIdx.x / TPR;
    const int col = (blockIdx.y * TPR + lane) * 8;
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = 0.f;
    if (col < a.N)
        for (int64_t j = c + 1 + g; j <= end; j += GB) {
            const Chunk<float> h = Chunk<float>::load(a.part + j * 2 * a.Np + col);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] += h.get(i);
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
// threads per row of the chunk-walking kernels
static int ltpr_for(int64_t N) {
    const int64_t nc = (N + 7) / 8;
    int l = 0;
    while (l < 8 && (int64_t(1) << l) < nc) ++l;
    return l;
}

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
    const int l = ltpr_for(a.N), rpb = 256 >> l;
    const int64_t g = std::min<int64_t>((a.M + rpb - 1) / rpb, 4096);
    return by_type(a.dtype, [&](auto ty) -> hipError_t {
        using T = decltype(ty);
        return launch(k_dropout<T>, dim3((unsigned)g), dim3(256), st, a.M, a.N, (const T*)a.x, a.ldx, (T*)a.y, a.ldy, l, k);
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
    const int l = ltpr_for(a.N), rpb = 256 >> l;
    const int64_t g = std::min<int64_t>((a.T + rpb - 1) / rpb, 4096);
    return by_type(a.dtype, [&](auto ty) -> hipError_t {
        return launch(k_emb_fwd<decltype(ty)>, dim3((unsigned)g), dim3(256), st, p, l);
    });
}

// the gradient's plan, a function of (T, N) alone: tokens per group and pieces
struct EmbPlan {
    int tpr, gb, tg, slices;
    int64_t pieces, tiles, Np;
    int64_t o_key[2], o_idx[2], o_hist, o_part, bytes;
};
static EmbPlan emb_plan(int64_t T, int64_t N) {
    EmbPlan q;
    q.Np = (N + 7) / 8 * 8;
    const int l = std::min(ltpr_for(N), 6);
    q.tpr = std::max(8, 1 << l);
    q.gb = 256 / q.tpr;
    q.slices = (int)((N + q.tpr * 8 - 1) / (q.tpr * 8));
    q.tg = T > 32768 ? 32 : 8;
    q.pieces = std::max<int64_t>(1, (T + (int64_t)q.gb * q.tg - 1) / ((int64_t)q.gb * q.tg));
    q.tiles = (T + RTILE - 1) / RTILE;
    int64_t o = 0;
    auto take = [&](int64_t b) {
        const int64_t at = o;
        o += (b + 255) / 256 * 256;
        return at;
    };
    for (int i = 0; i < 2; ++i) {
        q.o_key[i] = take(T * 4);
        q.o_idx[i] = take(T * 4);
    }
    q.o_hist = take((q.tiles + 1) * 256 * 4);
    q.o_part = take(q.pieces * 2 * q.Np * 4);
    q.bytes = o;
    return q;
}
int64_t emb_bwd_ws(int64_t T, int64_t N) { return emb_plan(T, N).bytes; }

__global__ __launch_bounds__(1024) void k_emb_clear(void* out, int64_t out_bytes) {
    fill_zero((uint32_t*)out, out_bytes / 4, (int64_t)blockIdx.x * 1024 + threadIdx.x, (int64_t)gridDim.x * 1024);
    if (blockIdx.x == 0 && threadIdx.x == 0 && (out_bytes & 2)) ((uint16_t*)out)[out_bytes / 2 - 1] = 0;
}

hipError_t emb_bwd(const mmvae_embedding_args& a, hipStream_t st) {
    const int64_t z = a.dtype == MMVAE_T_F32 ? 4 : 2, out_bytes = a.V * a.N * z;
    const int clear = (int)std::min<int64_t>((out_bytes / 4 + RTHR * 4 - 1) / (RTHR * 4) + 1, 1024);
    if (a.T == 0) return out_bytes ? launch(k_emb_clear, dim3((unsigned)clear), dim3(1024), st, a.dtable, out_bytes) : hipSuccess;
    const EmbPlan q = emb_plan(a.T, a.N);
    char* ws = (char*)a.ws;
    uint32_t* key[2] = {(uint32_t*)(ws + q.o_key[0]), (uint32_t*)(ws + q.o_key[1])};
    uint32_t* idx[2] = {(uint32_t*)(ws + q.o_idx[0]), (uint32_t*)(ws + q.o_idx[1])};
    uint32_t* hist = (uint32_t*)(ws + q.o_hist);
    const uint32_t V = (uint32_t)a.V;
    int passes = 1;
    while (passes < 4 && (V >> (8 * passes)) != 0) ++passes;
    int cur = 0;
    if (a.T <= RTILE) {
        OPCHK(launch(k_emb_sort1, dim3((unsigned)(1 + clear)), dim3(RTHR), st, a.ids, a.ids64, (int)a.T, V, passes, key[0], idx[0],
                     a.dtable, out_bytes));
    } else {
        const int tiles = (int)q.tiles, scanned = tiles > RFUSE ? 1 : 0;
        for (int p = 0; p < passes; ++p) {
            const uint32_t* ki = p ? key[cur] : nullptr;
            const uint32_t* xi = p ? idx[cur] : nullptr;
            const int nxt = p ? cur ^ 1 : 0;
            OPCHK(launch(k_emb_hist, dim3((unsigned)(tiles + (p ? 0 : clear))), dim3(RTHR), st, a.ids, a.ids64, ki, a.T, V, 8 * p, tiles,
                         hist, a.dtable, out_bytes));
            if (scanned) OPCHK(launch(k_emb_scan, dim3(256), dim3(256), st, tiles, hist));
            OPCHK(launch(k_emb_scatter, dim3((unsigned)tiles), dim3(RTHR), st, a.ids, a.ids64, ki, xi, a.T, V, 8 * p, tiles, scanned,
                         (const uint32_t*)hist, key[nxt], idx[nxt]));
            cur = nxt;
        }
    }
    EmbB b;
    b.T = a.T;
    b.N = (int)a.N;
    b.Np = q.Np;
    b.V = V;
    b.key = key[cur];
    b.idx = idx[cur];
    b.dy = a.dy;
    b.lddy = a.lddy;
    b.out = a.dtable;
    b.part = (float*)(ws + q.o_part);
    b.scale = a.scale;
    b.tg = q.tg;
    const dim3 grid((unsigned)q.pieces, (unsigned)q.slices), jgrid((unsigned)(q.pieces - 1), (unsigned)q.slices);
    return by_type(a.dtype, [&](auto ty) -> hipError_t {
        using T = decltype(ty);
        auto go = [&](auto t) -> hipError_t {
            OPCHK(launch(k_emb_seg<T, t.value>, grid, dim3(256), st, b));
            return q.pieces > 1 ? launch(k_emb_join<T, t.value>, jgrid, dim3(256), st, b, (int)q.pieces) : hipSuccess;
        };
        if (q.tpr == 8) return go(I<8>{});
        if (q.tpr == 16) return go(I<16>{});
        if (q.tpr == 32) return go(I<32>{});
        return go(I<64>{});
    });
}

// ---- argument checks: null, or what is wrong -------------------------------------------------
static bool type_ok(int t) { return t == MMVAE_T_F32 || t == MMVAE_T_BF16 || t == MMVAE_T_F16; }
static constexpr int64_t MAX_DIM = (int64_t(1) << 31) - 65536;  // rows, widths, tokens and table rows
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
    if (!bwd) {
        if (a.M > 0 && !a.y) return "y is null";
        if (!ld_ok(a.ldy, a.N, a.M)) return "y's row stride is below N";
        return nullptr;
    }
    if (a.M > 0 && (!a.dy || !a.mean || !a.rstd)) return "dy, mean or rstd is null";
    if (a.dx && !ld_ok(a.lddx, a.N, a.M)) return "dx's row stride is below N";
    if ((a.dw || a.db) && norm_bwd_ws(a.M, a.N) > 0 && (!a.ws || a.ws_bytes < norm_bwd_ws(a.M, a.N))) return "the workspace is below mmvae_layer_norm_bwd_ws(M, N) bytes";
    return nullptr;
}
const char* dropout_check(const mmvae_dropout_args& a) {
    if (a.M < 0 || a.N < 0 || a.M > MAX_DIM || a.N > MAX_DIM) return "need 0 <= M, N < 2^31";
    if (!type_ok(a.dtype)) return "types: f32, bf16 or f16";
    if (const char* m = drop_check(a.p)) return m;
    if (a.M > 0 && a.N > 0 && (!a.x || !a.y)) return "x or y is null";
    if (a.ldx < 0 || !ld_ok(a.ldy, a.N, a.M)) return "x's row stride is negative or y's below N";
    return nullptr;
}
const char* emb_check(const mmvae_embedding_args& a, bool bwd) {
    if (a.T < 0 || a.N < 1 || a.V < 0 || a.T > MAX_DIM || a.N >= (1 << 24) || a.V > MAX_DIM)
        return "need 0 <= T, V < 2^31 and 1 <= N < 2^24";
    if (!type_ok(a.dtype)) return "types: f32, bf16 or f16";
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
    if (a.T > 0 && (!a.ws || a.ws_bytes < emb_bwd_ws(a.T, a.N))) return "the workspace is below mmvae_embedding_bwd_ws(T, N) bytes";
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
int64_t mmvae_embedding_bwd_ws(int64_t T, int64_t N) { return T < 0 || N < 1 ? 0 : emb_bwd_ws(T, N); }

}  // extern "C"
