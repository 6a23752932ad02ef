// Layer norm, forward and backward (ops.hip's entries): the kernels and their launch for one type of
// activations; each type is a translation unit of its own (norm_f32 / _bf16 / _f16.hip).
#pragma once
#include "ops_dev.hpp"

namespace mmvae {

// =======================================================================================
// Layer norm over rows of N: y = drop(act(xh w + b)), xh = (x - mean) rstd
// TPR threads hold a row (VPT chunks each) in registers: x is read once, the variance is the
// mean square of the differences from the mean (two dependent sums, but no cancellation).
//
// Both directions are bound by memory where rows are many: forward reads x and writes y, backward
// reads x and dy and writes dx; the row sums between a row's loads and its stores are hidden by
// other rows' waves, or by the next row's loads where a row fills the workgroup.  Measured:
//                       forward                backward
//   32768 x 1024 bf16   29.8 us, 4.5 TB/s      44.4 us, 4.5 TB/s   (with dropout)
//   4096 x 20000 bf16   68 us,   4.8 TB/s      123 us,  4.0 TB/s
//   4096 x 128 f32      4.2 us                 4.7 us              (with dropout)
//   100 x 48 f32        2.7 us                 3.7 us              (a launch's time)
// against 5.1 TB/s of a large copy.  The backward of long rows is the furthest off: its column sums
// (16 registers a chunk) leave room for two rows in flight in 8 waves of a CU.
// =======================================================================================
struct NormP {
    int64_t M;
    int N;
    const void *x, *w, *b, *dy;
    int64_t ldx, lddy, ldy;  // ldy: of y, or of dx
    void* y;                 // y, or dx
    float *mean, *rstd;
    float* part;             // backward: the workgroups' sums [grid][2][Np], or null
    void *dw, *db;           // written by the strips
    int64_t Np;
    float eps;
    int relu;
    bool wf32;
    bool b_lds;              // forward, weights in LDS: the biases too
    int strips, strip_waves; // backward: the first workgroups sum dw and db in strips of 8 columns, so many waves each
    DropKey drop;
};

// A row's statistics, and xh and u = xh w + b as forward and backward both compute them (the ReLU's side
// must be the same): xh from the difference, exact near the mean.  w and b come multiplied by the dropout factor
// (a ReLU commutes with it).  The mean is a quotient: a product, sum (1 / N), goes into the difference unrounded
// (one fma), and the forward's u is then not that of the stored mean; and a row of one value is off by its last bit
// times rstd, up to 1 / sqrt(eps).  For 16-bit values too, whose rows often hold few different values (as x r - m r
// with a product for m, constant rows of 5000 missed the bias by 0.1): 65536 x 128 bf16 forward 6.9 -> 7.2 us, 32768 x
// 517 f16 backward 37.0 -> 38.3, elsewhere up to 1 %.
struct RowStat {
    float mean, rstd;
    MMVAE_DEV void set(float m, float r) {
        mean = m;
        rstd = r;
    }
    MMVAE_DEV float xh(float x) const { return (x - mean) * rstd; }
    MMVAE_DEV float u(float x, float w, float b) const { return __builtin_fmaf(xh(x), w, b); }
};
// 8 weights times the factor
template <class T> MMVAE_DEV void ldws(const void* w, bool f32, int col, int n, float none, float s, float v[8]) {
    ldw<T>(w, f32, col, n, none, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= s;
}

// How a thread keeps its row and weights, by the 256 registers that a wave has at up to 512 threads (with fewer
// threads a row other rows' waves hide the loads too):
//   HOLD  the weights in registers over all rows, else in LDS (16 V of w and b forward, 8 V of w backward);
//   PRE   the next row's loads in flight under this row's sums;
//   AGAIN (backward) x and dy read in both phases, where they do not fit beside the 16 V column sums.
// ROOM: what is left beside temporaries, as the compiler uses them (no variant that is launched spills
// more than a few registers).
template <class T, int VPT, int BLK, bool MASK, bool EVEN> struct LnKeep {
    static_assert(BLK <= 512, "256 registers a lane");
    static constexpr int X = (int)sizeof(T) * 2;  // registers of a chunk
    static constexpr int ROOM = 256 - 66 - (MASK ? 10 : 0) - (EVEN ? 0 : 14);
    static constexpr int B = 16 + (MASK ? 12 : 0);  // a chunk's column sums (and masks)
    static constexpr bool F_HOLD = (16 + X) * VPT <= ROOM;
    static constexpr bool F_PRE = ((F_HOLD ? 16 : 0) + 2 * X) * VPT <= ROOM;
    static constexpr bool B_AGAIN = (B + 2 * X) * VPT > ROOM;
    static constexpr bool B_PRE = !B_AGAIN && (B + 4 * X) * VPT <= ROOM;
    static constexpr bool B_HOLD = !B_AGAIN && (B + (B_PRE ? 4 : 2) * X + 8) * VPT <= ROOM;
};

static constexpr int LN_LDS = 163840;  // bytes of LDS of a CU

// a pointer into LDS that the compiler takes for a new one: what is read there is read again (with every
// row, in every phase) instead of being kept in registers from before
MMVAE_DEV float* lds_anew(float* l) {
    int zero = 0;
    asm volatile("" : "+s"(zero));
    return l + zero;
}

// forward.  MASK: with a ReLU or dropout (dropout adds 2.5 us at 32768 x 1024 bf16); EVEN: N a multiple of 8, whose
// loads and stores need no tail (and no branch)
template <class T, int TPR, int VPT, int BLK, bool MASK, bool EVEN>
__global__ __launch_bounds__(BLK) void k_ln_fwd(NormP a) {
    constexpr int RPB = BLK / TPR;
    typedef LnKeep<T, VPT, BLK, MASK, EVEN> Keep;
    constexpr bool HOLD = Keep::F_HOLD, PRE = Keep::F_PRE;
    extern __shared__ float4 dyn_lds[];
    float* lw = reinterpret_cast<float*>(dyn_lds);
    __shared__ float red[2][BLK / 64];
    const int lane = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    const int N = a.N, slots = (N + 7) / 8;
    const float inv = 1.f / (float)N, sc = MASK && a.drop.thr ? a.drop.s : 1.f;
    if (MASK) drop_state(a.drop);
    float hw[HOLD ? VPT : 1][8], hb[HOLD ? VPT : 1][8];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int c = j * TPR + lane, col = c * 8;
        ldws<T>(a.w, a.wf32, col, N - col, 1.f, sc, hw[HOLD ? j : 0]);
        if (HOLD || a.b_lds) ldws<T>(a.b, a.wf32, col, N - col, 0.f, sc, hb[HOLD ? j : 0]);
        if (!HOLD && c < slots) {
            lds_put8(lw, slots, c, hw[0]);
            if (a.b_lds) lds_put8(lw + slots * 8, slots, c, hb[0]);
        }
    }
    const int64_t step = (int64_t)gridDim.x * RPB;
    Chunk<T> xc[VPT], xn[PRE ? VPT : 1];
    auto fetch = [&](int64_t r, Chunk<T>* x) {
        const T* xr = (const T*)a.x + (r < a.M ? r : 0) * a.ldx;
#pragma unroll
        for (int j = 0; j < VPT; ++j) x[j] = ld_row<EVEN>(xr, (j * TPR + lane) * 8, N);
    };
    if constexpr (PRE) fetch((int64_t)blockIdx.x * RPB + grp, xn);
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.M; r0 += step) {
        const int64_t row = r0 + grp;
        const bool ok = row < a.M;
        float s = 0.f;
        if constexpr (PRE) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) xc[j] = xn[j];
            if (r0 + step < a.M) fetch(row + step, xn);
        } else {
            fetch(row, xc);
        }
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            float t = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) t += xc[j].get(i);
            s += !EVEN || (j * TPR + lane) * 8 < N ? t : 0.f;
        }
        const float mean = row_sum<TPR>(s, red[0]) / (float)N;
        float q = 0.f;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int n = N - (j * TPR + lane) * 8;
            float t = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = EVEN || i < n ? xc[j].get(i) - mean : 0.f;
                t = __builtin_fmaf(d, d, t);
            }
            q += !EVEN || n > 0 ? t : 0.f;
        }
        RowStat st;
        st.set(mean, 1.f / sqrtf(row_sum<TPR>(q, red[1]) * inv + a.eps));
        if (ok) {
            T* yr = (T*)a.y + row * a.ldy;
            const float* rw = HOLD ? lw : lds_anew(lw);
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const int c = j * TPR + lane, col = c * 8, n = N - col;
                if (n <= 0) continue;
                float w[8], b[8];
                if constexpr (!HOLD) {
                    lds_get8(rw, slots, c, w);
                    if (a.b_lds) lds_get8(rw + slots * 8, slots, c, b);
                    else ldws<T>(a.b, a.wf32, col, n, 0.f, sc, b);
                }
                float u[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    u[i] = st.u(xc[j].get(i), HOLD ? hw[HOLD ? j : 0][i] : w[i], HOLD ? hb[HOLD ? j : 0][i] : b[i]);
                if (MASK && a.relu) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) u[i] = u[i] > 0.f || u[i] != u[i] ? u[i] : 0.f;  // (a NaN stays one)
                }
                if (MASK && a.drop.thr) {
                    bool kept[8];
                    keep8(a.drop, row, c, kept);
#pragma unroll
                    for (int i = 0; i < 8; ++i) u[i] = kept[i] ? u[i] : 0.f;
                }
                Chunk<T> yc;
#pragma unroll
                for (int i = 0; i < 8; ++i) yc.set(i, u[i]);
                if constexpr (EVEN) yc.store(yr + col);
                else st8(yr + col, n, yc);
            }
            if (lane == 0) {
                if (a.mean) a.mean[row] = mean;
                if (a.rstd) a.rstd[row] = st.rstd;
            }
        }
        if constexpr (TPR > 64) __syncthreads();  // the next row's sums reuse `red`
    }
}

// strips of 8 columns summed over all rows: the row statistics are inputs, so this needs nothing of what the
// row workgroups do.  A workgroup's 8 waves sum one strip, or (rows above 4096 columns, where strips are many)
// four strips: lane sums in each wave, then a strip's waves in order (256 x 20000 bf16, waves a strip: 8 24
// us, 4 17.9, 2 16.8, 1 16.7; 512 rows with dropout: 4 39.9, 2 38.1, 1 39.8).
static constexpr int STRIP_BLK = 512;
template <class T, bool MASK, bool EVEN> MMVAE_DEV void ln_strip(const NormP& a, float ds) {
    __shared__ float sh[STRIP_BLK / 64][17];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, sw = a.strip_waves, each = STRIP_BLK / 64 / sw;
    // (workgroups go round the 8 XCDs: neighbouring strips, which share cache lines, to the same one)
    const int c0 = ((int)(blockIdx.x & 7) * (a.strips >> 3) + (int)(blockIdx.x >> 3)) * each;
    const int c = c0 + wave / sw, col = c * 8, N = a.N, n = N - col;
    float w[8], b[8], aw[8] = {}, ab[8] = {};
    if (MASK) {
        ldws<T>(a.w, a.wf32, col, n, 1.f, ds, w);
        ldws<T>(a.b, a.wf32, col, n, 0.f, ds, b);
    }
    const int64_t step = 64 * sw;
    for (int64_t r0 = (wave % sw) * 64 + lane; r0 < a.M && n > 0; r0 += 2 * step) {  // two rows at once
        Chunk<T> x[2], d[2];
        RowStat st[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int64_t row = r0 + step * k, rr = row < a.M ? row : r0;
            x[k] = ld_row<EVEN>((const T*)a.x + rr * a.ldx, col, N);
            d[k] = ld_row<EVEN>((const T*)a.dy + rr * a.lddy, col, N);
            st[k].set(a.mean[rr], a.rstd[rr]);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int64_t row = r0 + step * k;
            if (row >= a.M) break;
            if (MASK) {
                bool on[8] = {true, true, true, true, true, true, true, true};
                if (a.drop.thr) keep8(a.drop, row, c, on);
                if (a.relu) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) on[i] = on[i] && st[k].u(x[k].get(i), w[i], b[i]) > 0.f;
                }
                d[k].keep(on);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = d[k].get(i);
                aw[i] = __builtin_fmaf(v, st[k].xh(x[k].get(i)), aw[i]);
                ab[i] += v;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float s = lanes_sum<64>(aw[i]), t = lanes_sum<64>(ab[i]);
        if (lane == 0) {
            sh[wave][i] = s;
            sh[wave][8 + i] = t;
        }
    }
    __syncthreads();
    const int k = threadIdx.x & 15, q0 = threadIdx.x >> 4, at = (c0 + q0) * 8 + (k & 7);
    void* o = k < 8 ? a.dw : a.db;
    if (q0 >= each || at >= N || !o) return;
    float v = 0.f;
    for (int q = q0 * sw; q < (q0 + 1) * sw; ++q) v += sh[q][k];
    if (MASK) v *= ds;
    if (a.wf32) ((float*)o)[at] = v;
    else ((T*)o)[at] = (T)v;
}
// the strips alone: of rows that are read in sweeps, and where dx overwrites dy or x
template <class T, bool MASK, bool EVEN> __global__ __launch_bounds__(STRIP_BLK) void k_ln_strips(NormP a) {
    if (MASK) drop_state(a.drop);
    ln_strip<T, MASK, EVEN>(a, MASK && a.drop.thr ? a.drop.s : 1.f);
}

// backward: du = dy m [u > 0], g = du w, dx = rstd (g - mean(g) - xh mean(g xh)); the workgroup's
// sums of du xh and du over its rows (of the unscaled du: times the dropout factor once, at the end; fixed
// order: a thread's rows, then the row groups) -> part, if there is one.  The masks are recomputed and folded
// into dy, the dropout factor into the weights, and dx is one linear form of dy and x, so that a row costs
// two fma an element beside its sums (32768 x 1024 bf16 with dropout: 49.1 -> 44.0 us).  Elements behind a
// row's end are loaded as 0 and add 0.
template <class T, int TPR, int VPT, int BLK, bool MASK, bool EVEN>
__global__ __launch_bounds__(BLK, BLK / 256) void k_ln_bwd(NormP a) {
    constexpr int RPB = BLK / TPR;
    typedef LnKeep<T, VPT, BLK, MASK, EVEN> Keep;
    constexpr bool HOLD = Keep::B_HOLD, AGAIN = Keep::B_AGAIN, PRE = Keep::B_PRE;
    extern __shared__ float4 dyn_lds[];
    float* lw = reinterpret_cast<float*>(dyn_lds);
    __shared__ float red[2][BLK / 64];
    const int lane = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    const int N = a.N, slots = (N + 7) / 8;
    const float inv = 1.f / (float)N, ds = MASK && a.drop.thr ? a.drop.s : 1.f;
    if (MASK) drop_state(a.drop);
    int strips = 0;
    if constexpr (BLK == STRIP_BLK) {
        strips = a.strips;
        if ((int)blockIdx.x < strips) return ln_strip<T, MASK, EVEN>(a, ds);
    }
    const int64_t first = (int64_t)((int)blockIdx.x - strips) * RPB;
    float hw[HOLD ? VPT : 1][8];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int c = j * TPR + lane, col = c * 8;
        ldws<T>(a.w, a.wf32, col, N - col, 1.f, ds, hw[HOLD ? j : 0]);
        if (!HOLD && c < slots) lds_put8(lw, slots, c, hw[0]);
    }
    float aw[VPT][8], ab[VPT][8];
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) aw[j][i] = ab[j][i] = 0.f;
    // a row's x and dy, dy without what dropout and ReLU take away: du = ds dc, g = dc (ds w).  (AGAIN: each phase reads
    // them, the second with the first's bits)
    const int64_t step = (int64_t)((int)gridDim.x - strips) * RPB;
    Chunk<T> xc[AGAIN ? 1 : VPT], dc[AGAIN ? 1 : VPT], xn[PRE ? VPT : 1], dn[PRE ? VPT : 1];
    uint32_t bits[VPT];
    float mean = 0.f, rstd = 0.f, mean_n = 0.f, rstd_n = 0.f;
    auto read = [&](int64_t r, int j, Chunk<T>& x, Chunk<T>& d) {
        const int col = (j * TPR + lane) * 8;
        const bool ok = r < a.M;
        x = ld_row<EVEN>((const T*)a.x + (ok ? r : 0) * a.ldx, col, N);
        d = ld_row<EVEN>((const T*)a.dy + (ok ? r : 0) * a.lddy, col, N);
    };
    auto fetch = [&](int64_t r, Chunk<T>* x, Chunk<T>* d, float& m, float& s) {
        m = r < a.M ? a.mean[r] : 0.f;
        s = r < a.M ? a.rstd[r] : 0.f;
        if constexpr (!AGAIN) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) read(r, j, x[j], d[j]);
        }
    };
    if constexpr (PRE) fetch(first + grp, xn, dn, mean_n, rstd_n);
    for (int64_t r0 = first; r0 < a.M; r0 += step) {
        const int64_t row = r0 + grp;
        const bool ok = row < a.M;
        if constexpr (PRE) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                xc[j] = xn[j];
                dc[j] = dn[j];
            }
            mean = mean_n;
            rstd = rstd_n;
            if (r0 + step < a.M) fetch(row + step, xn, dn, mean_n, rstd_n);
        } else {
            fetch(row, xc, dc, mean, rstd);
        }
        RowStat st;
        st.set(mean, rstd);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int c = j * TPR + lane, col = c * 8, n = N - col;
            Chunk<T>&x = xc[AGAIN ? 0 : j], &dd = dc[AGAIN ? 0 : j];
            if constexpr (AGAIN) read(row, j, x, dd);
            if ((EVEN && col >= N) || !ok) dd = Chunk<T>{};  // adds nothing
            float w[8], b[8];
            if constexpr (HOLD) {
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = hw[HOLD ? j : 0][i];
            } else {
                // (a chunk behind the row's end multiplies zeros, by a slot that this thread wrote itself: another wave's
                // may not be there yet, and what an earlier kernel left in LDS can be a NaN)
                static_assert(VPT > 1, "the thread's first slot is in the row");
                lds_get8(lds_anew(lw), slots, c < slots ? c : lane, w);
            }
            if (MASK) {
                bool on[8] = {true, true, true, true, true, true, true, true};
                if (a.drop.thr) keep8(a.drop, row, c, on);
                if (a.relu) {
                    ldws<T>(a.b, a.wf32, col, n, 0.f, ds, b);
#pragma unroll
                    for (int i = 0; i < 8; ++i) on[i] = on[i] && st.u(x.get(i), w[i], b[i]) > 0.f;
                }
                dd.keep(on);
                if constexpr (AGAIN) {
                    bits[j] = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) bits[j] |= on[i] ? 1u << i : 0u;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = dd.get(i), dxh = d * st.xh(x.get(i));
                aw[j][i] += dxh;
                ab[j][i] += d;
                s1 = __builtin_fmaf(d, w[i], s1);
                s2 = __builtin_fmaf(dxh, w[i], s2);
            }
            // chunk by chunk, each sum taken here: the products of all chunks at once, kept for sums further
            // down, would not fit the registers
            if constexpr (VPT > 1) {
#pragma unroll
                for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(aw[j][i]), "+v"(ab[j][i]));
                asm volatile("" : "+v"(s1), "+v"(s2));
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (a.y) {
            if constexpr (VPT > 1 && !AGAIN) {
#pragma unroll
                for (int j = 0; j < VPT; ++j) {
                    xc[j].anew();
                    dc[j].anew();
                }
            }
            const float c1 = row_sum<TPR>(s1, red[0]) * inv, c2 = row_sum<TPR>(s2, red[1]) * inv;
            // dx = d (w rstd) + x A + B: the row's part, - rstd (c1 + xh c2), is linear in x
            const float A = -rstd * rstd * c2, B = -rstd * c1 - mean * A;
            if (ok) {
                T* yr = (T*)a.y + row * a.ldy;
#pragma unroll
                for (int j = 0; j < VPT; ++j) {
                    const int col = (j * TPR + lane) * 8, n = N - col;
                    if (n <= 0) continue;
                    if constexpr (AGAIN) {
                        read(row, j, xc[0], dc[0]);
                        bool on[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) on[i] = (bits[j] >> i) & 1;
                        if (MASK) dc[0].keep(on);
                    }
                    const Chunk<T>&x = xc[AGAIN ? 0 : j], &dd = dc[AGAIN ? 0 : j];
                    float w[8];
                    if constexpr (HOLD) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) w[i] = hw[HOLD ? j : 0][i];
                    } else {
                        lds_get8(lds_anew(lw), slots, j * TPR + lane, w);
                    }
                    Chunk<T> o;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float r = sizeof(T) == 4 ? __builtin_fmaf(x.get(i) - mean, A, -rstd * c1) : __builtin_fmaf(x.get(i), A, B);
                        o.set(i, __builtin_fmaf(dd.get(i), w[i] * rstd, r));
                    }
                    if constexpr (EVEN) o.store(yr + col);
                    else st8(yr + col, n, o);
                    if constexpr (VPT > 1) __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        if constexpr (TPR > 64) __syncthreads();
    }
    if (!a.part) return;
    auto put = [&](int h, int c, float v) { a.part[((int64_t)((int)blockIdx.x - strips) * 2 + h) * a.Np + c] = MASK ? v * ds : v; };
    if constexpr (RPB == 1) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int col = (j * TPR + lane) * 8;
            if (col < N) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {  // (Np is a multiple of 8)
                    put(0, col + i, aw[j][i]);
                    put(1, col + i, ab[j][i]);
                }
            }
        }
    } else {
        __shared__ float sh[RPB][TPR * VPT * 8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < VPT; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) sh[grp][(j * TPR + lane) * 8 + i] = h ? ab[j][i] : aw[j][i];
            __syncthreads();
            for (int c = threadIdx.x; c < TPR * VPT * 8; c += BLK) {
                float t = 0.f;
#pragma unroll 8
                for (int g = 0; g < RPB; ++g) t += sh[g][c];
                if (c < a.Np) put(h, c, t);
            }
        }
    }
}

// dw / db: the G partial rows of a column summed in a fixed order (workgroup: 32 columns x 32 row
// groups, a group's loads four at a time).  256 x 2 x 20000 sums (41 MB) 9.7 us, 4.2 TB/s; 512 x 2 x 1024
// 4.8 us, of which 2.5 are a launch's
template <class W>
__global__ __launch_bounds__(1024) void k_ln_wred(int N, int64_t Np, int G, const float* __restrict__ part, W* __restrict__ dw,
                                                  W* __restrict__ db) {
    __shared__ float sh[32][33];
    const int lane = threadIdx.x & 31, g0 = threadIdx.x >> 5;
    const int64_t col = (int64_t)blockIdx.x * 32 + lane;  // of [2][Np]
    const int64_t cc = col < 2 * Np ? col : 0;
    float t = 0.f;
    for (int g = g0; g < G; g += 128) {
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = part[(int64_t)min(g + 32 * k, G - 1) * 2 * Np + cc];
#pragma unroll
        for (int k = 0; k < 4; ++k) t += g + 32 * k < G ? v[k] : 0.f;
    }
    sh[g0][lane] = t;
    __syncthreads();
    if (threadIdx.x < 32 && col < 2 * Np) {
        t = 0.f;
#pragma unroll
        for (int g = 0; g < 32; ++g) t += sh[g][lane];
        const bool second = col >= Np;
        const int64_t c = second ? col - Np : col;
        W* o = second ? db : dw;
        if (o && c < N) o[c] = (W)t;
    }
}

// Rows too long for the registers (N > 32,768): each sweep reads the row again, from the last-level cache
// where it fits (2048 x 40000 bf16: forward 104 us, 3.1 TB/s of x and y; backward 235 us).  32768 / 32776 columns
// of 4096 bf16 rows: forward 102 / 187 us, backward 265 / 386.
static constexpr int LONG_N = 32768;
template <class T> __global__ __launch_bounds__(1024) void k_ln_fwd_long(NormP a) {
    __shared__ float red[2][16];
    const int N = a.N;
    const float inv = 1.f / (float)N, sc = a.drop.thr ? a.drop.s : 1.f;
    drop_state(a.drop);
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        const T* xr = (const T*)a.x + row * a.ldx;
        float s = 0.f;
        for (int64_t col = threadIdx.x * 8; col < N; col += 8192) {
            const Chunk<T> c = ld8(xr + col, (int)(N - col));
            float t = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) t += c.get(i);
            s += t;
        }
        const float mean = row_sum<1024>(s, red[0]) / (float)N;
        float q = 0.f;
        for (int64_t col = threadIdx.x * 8; col < N; col += 8192) {
            const int n = (int)(N - col);
            const Chunk<T> c = ld8(xr + col, n);
            float t = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = c.get(i) - mean;
                t += i < n ? d * d : 0.f;
            }
            q += t;
        }
        RowStat st;
        st.set(mean, 1.f / sqrtf(row_sum<1024>(q, red[1]) * inv + a.eps));
        T* yr = (T*)a.y + row * a.ldy;
        for (int64_t col = threadIdx.x * 8; col < N; col += 8192) {
            const int n = (int)(N - col);
            const Chunk<T> c = ld8(xr + col, n);
            float w[8], b[8];
            bool kept[8];
            ldws<T>(a.w, a.wf32, (int)col, n, 1.f, sc, w);
            ldws<T>(a.b, a.wf32, (int)col, n, 0.f, sc, b);
            if (a.drop.thr) keep8(a.drop, row, (int)(col >> 3), kept);
            Chunk<T> yc;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float u = st.u(c.get(i), w[i], b[i]);
                if (a.relu) u = u > 0.f || u != u ? u : 0.f;
                if (a.drop.thr) u = kept[i] ? u : 0.f;
                yc.set(i, u);
            }
            st8(yr + col, n, yc);
        }
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = st.rstd;
        }
        __syncthreads();
    }
}
// one chunk's dy without what dropout and ReLU take away, xh, and the weights times the dropout factor
template <class T>
MMVAE_DEV void ln_du(const NormP& a, int64_t row, int64_t col, const RowStat& st, float w[8], float du[8], float xh[8]) {
    const int n = (int)(a.N - col);
    const Chunk<T> xc = ld8((const T*)a.x + row * a.ldx + col, n), dc = ld8((const T*)a.dy + row * a.lddy + col, n);
    const float sc = a.drop.thr ? a.drop.s : 1.f;
    float b[8];
    bool kept[8];
    ldws<T>(a.w, a.wf32, (int)col, n, 1.f, sc, w);
    if (a.relu) ldws<T>(a.b, a.wf32, (int)col, n, 0.f, sc, b);
    if (a.drop.thr) keep8(a.drop, row, (int)(col >> 3), kept);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        xh[i] = i < n ? st.xh(xc.get(i)) : 0.f;
        float d = dc.get(i);
        if (a.drop.thr) d = kept[i] ? d : 0.f;
        if (a.relu) d = st.u(xc.get(i), w[i], b[i]) > 0.f ? d : 0.f;
        du[i] = i < n ? d : 0.f;
    }
}
template <class T> __global__ __launch_bounds__(1024) void k_ln_bwd_long(NormP a) {
    __shared__ float red[2][16];
    const float inv = 1.f / (float)a.N;
    drop_state(a.drop);
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        RowStat st;
        st.set(a.mean[row], a.rstd[row]);
        float s1 = 0.f, s2 = 0.f, w[8], du[8], xh[8];
        for (int64_t col = threadIdx.x * 8; col < a.N; col += 8192) {
            ln_du<T>(a, row, col, st, w, du, xh);
            float t1 = 0.f, t2 = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                t1 = __builtin_fmaf(du[i], w[i], t1);
                t2 = __builtin_fmaf(du[i] * xh[i], w[i], t2);
            }
            s1 += t1;
            s2 += t2;
        }
        const float c1 = row_sum<1024>(s1, red[0]) * inv, c2 = row_sum<1024>(s2, red[1]) * inv;
        T* yr = (T*)a.y + row * a.ldy;
        for (int64_t col = threadIdx.x * 8; col < a.N; col += 8192) {
            ln_du<T>(a, row, col, st, w, du, xh);
            Chunk<T> o;
#pragma unroll
            for (int i = 0; i < 8; ++i) o.set(i, st.rstd * (__builtin_fmaf(du[i], w[i], -c1) - xh[i] * c2));
            st8(yr + col, (int)(a.N - col), o);
        }
        __syncthreads();
    }
}
// their weight gradients: thread = a chunk of columns, workgroup row y = a stripe of rows
template <class T> __global__ __launch_bounds__(256) void k_ln_cols(NormP a) {
    const int64_t col = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (col >= a.N) return;
    drop_state(a.drop);
    float aw[8] = {}, ab[8] = {}, w[8], du[8], xh[8];
    for (int64_t row = blockIdx.y; row < a.M; row += gridDim.y) {
        RowStat st;
        st.set(a.mean[row], a.rstd[row]);
        ln_du<T>(a, row, col, st, w, du, xh);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            aw[i] += du[i] * xh[i];
            ab[i] += du[i];
        }
    }
    float* pw = a.part + (int64_t)blockIdx.y * 2 * a.Np;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        pw[col + i] = a.drop.thr ? aw[i] * a.drop.s : aw[i];
        pw[a.Np + col + i] = a.drop.thr ? ab[i] * a.drop.s : ab[i];
    }
}

// =======================================================================================
// Host side
// =======================================================================================
// the row layout by width: threads per row, chunks per thread, threads per workgroup.  Up to 64 lanes a
// row stays inside a wave and needs no barrier; above 8192 columns 512 threads with 256 registers each keep
// the next row's loads in flight, which 1024 threads with 128 do not (4096 x 20000 bf16 forward 72 -> 67 us).
template <class F> inline hipError_t by_width(int N, F&& f) {
    const int nc = (N + 7) / 8;
    if (nc <= 8) return f(I<8>{}, I<1>{}, I<256>{});
    if (nc <= 16) return f(I<16>{}, I<1>{}, I<256>{});
    if (nc <= 32) return f(I<32>{}, I<1>{}, I<256>{});
    if (nc <= 64) return f(I<64>{}, I<1>{}, I<256>{});
    if (nc <= 128) return f(I<64>{}, I<2>{}, I<256>{});
    if (nc <= 256) return f(I<256>{}, I<1>{}, I<256>{});
    if (nc <= 512) return f(I<256>{}, I<2>{}, I<256>{});
    if (nc <= 512 * 2) return f(I<512>{}, I<2>{}, I<512>{});
    if (nc <= 512 * 3) return f(I<512>{}, I<3>{}, I<512>{});
    if (nc <= 512 * 4) return f(I<512>{}, I<4>{}, I<512>{});
    if (nc <= 512 * 5) return f(I<512>{}, I<5>{}, I<512>{});
    if (nc <= 512 * 6) return f(I<512>{}, I<6>{}, I<512>{});
    return f(I<512>{}, I<8>{}, I<512>{});
}
// The backward's own: rows of 3521 .. 4096 on 512 threads, so that as many waves leave half the partial
// sums (4096 x 4096 bf16 31.4 -> 26.0 us; at 3300 columns the idle lanes cost more, 8192 rows 49 -> 56 us)
constexpr int HALF_N = 3520;
template <class F> inline hipError_t by_width_bwd(int N, F&& f) {
    return N > HALF_N && N <= 4096 ? f(I<512>{}, I<1>{}, I<512>{}) : by_width(N, f);
}
// Backward with masks: above 20,480 columns the sums do not stay in the registers (228 bytes a lane spilled), and the
// rows are read in sweeps.  Dropout, us, 20480 / 20488 columns: 100 rows bf16 14.9 / 18.3, 512 36 / 40, 2048 92 / 125, 4096
// 145 / 264 (f32 262 / 415); without masks 4096 rows 127 / 133.
constexpr int LONG_PARTS = 128, FITS_N = 20480, STRIP_N = 4096;
// A backward of few rows sums dw and db in strips of columns, beside the row workgroups of the same launch: x
// and dy are read a second time, but there are no partial sums to write, read and add up.  us of both ways
// (bf16, calls back to back): 100 x 128 2.6 / 5.2, 1024 x 1024 4.7 / 7.6, 1024 x 4096 11.2 / 25.1, 100 x 20000
// 10.2 / 34.6, 512 x 20000 27.5 / 48.0; past the limits the second reading costs more: 4096 x 128 6.4 / 5.9,
// 4096 x 1024 13.0 / 11.5, 1024 x 16800 with dropout 57 / 57.
inline bool norm_strips(int64_t M, int64_t N) { return N <= STRIP_N ? M <= 2048 && M * N <= (1 << 22) : M <= 512; }
template <class F> inline hipError_t by_width_strips(int N, F&& f) {
    const int nc = (N + 7) / 8;
    if (nc <= 8) return f(I<8>{}, I<1>{}, I<STRIP_BLK>{});
    if (nc <= 16) return f(I<16>{}, I<1>{}, I<STRIP_BLK>{});
    if (nc <= 32) return f(I<32>{}, I<1>{}, I<STRIP_BLK>{});
    if (nc <= 64) return f(I<64>{}, I<1>{}, I<STRIP_BLK>{});
    if (nc <= 128) return f(I<64>{}, I<2>{}, I<STRIP_BLK>{});
    if (nc <= 512) return f(I<512>{}, I<1>{}, I<STRIP_BLK>{});
    return by_width(N, f);
}
inline NormP norm_p(const mmvae_norm_args& a) {
    NormP p;
    std::memset(&p, 0, sizeof(p));
    p.M = a.M;
    p.N = (int)a.N;
    p.x = a.x;
    p.ldx = a.ldx;
    p.w = a.w;
    p.b = a.b;
    p.mean = a.mean;
    p.rstd = a.rstd;
    p.eps = a.eps;
    p.relu = a.relu;
    p.wf32 = a.wtype == MMVAE_T_F32;
    p.Np = (a.N + 7) / 8 * 8;
    p.drop = drop_key(a.p, a.seed, a.step, a.row_offset, a.state);
    return p;
}
inline int norm_rpb(int64_t N) {  // rows a workgroup holds at once
    int r = 1;
    (void)by_width((int)std::min<int64_t>(N, LONG_N), [&](auto t, auto, auto b) {
        r = b.value / t.value;
        return hipSuccess;
    });
    return r;
}
// Workgroups of the backward = rows of partial sums: two workgroups of 256 threads a CU, or one of 512.  More
// of them hide more of the loads' time, but write and read more sums (bf16: 4096 x 8192 512 parts 58 us, 256
// 49 us; 32768 x 1024 256 parts 51 us, 512 47 us).
inline int64_t norm_parts(int64_t M, int64_t N) {
    if (N > LONG_N) return std::min<int64_t>(M, LONG_PARTS);
    const int64_t need = (M + norm_rpb(N) - 1) / norm_rpb(N);
    return std::min<int64_t>(need, N > HALF_N ? 256 : 512);
}
inline int64_t norm_ws_bytes(int64_t M, int64_t N) {
    if (norm_strips(M, N)) return 0;
    return norm_parts(std::max<int64_t>(M, 1), N) * 2 * ((N + 7) / 8 * 8) * (int64_t)sizeof(float);
}

// with a ReLU or dropout; N a multiple of the chunk
template <class F> inline hipError_t by_flags(const NormP& p, F&& f) {
    const bool m = p.relu || p.drop.thr, e = p.N % 8 == 0;
    if (m) return e ? f(std::true_type{}, std::true_type{}) : f(std::true_type{}, std::false_type{});
    return e ? f(std::false_type{}, std::true_type{}) : f(std::false_type{}, std::false_type{});
}

template <class T> hipError_t norm_fwd_t(const mmvae_norm_args& a, hipStream_t st) {
    NormP p = norm_p(a);
    p.y = a.y;
    p.ldy = a.ldy;
    if (a.N > LONG_N) return launch(k_ln_fwd_long<T>, dim3((unsigned)std::min<int64_t>(a.M, 512)), dim3(1024), st, p);
    return by_width(p.N, [&](auto t, auto v, auto b) -> hipError_t {
        constexpr int RPB = b.value / t.value;
        const int64_t g = std::min<int64_t>((a.M + RPB - 1) / RPB, 256 * (2048 / b.value));
        return by_flags(p, [&](auto m, auto e) {
            size_t lds = 0;
            if (!LnKeep<T, v.value, b.value, m.value, e.value>::F_HOLD) {
                p.b_lds = 2 * p.Np * 4 <= LN_LDS - 256;  // (beside the waves' sums)
                lds = (p.b_lds ? 2 : 1) * (size_t)p.Np * 4;
            }
            return launch_lds(lds, k_ln_fwd<T, t.value, v.value, b.value, m.value, e.value>, dim3((unsigned)g), dim3(b.value), st, p);
        });
    });
}

template <class T> hipError_t norm_bwd_t(const mmvae_norm_args& a, hipStream_t st) {
    NormP p = norm_p(a);
    p.dy = a.dy;
    p.lddy = a.lddy;
    p.y = a.dx;
    p.ldy = a.lddx;
    const bool wg = a.dw || a.db, strips = wg && norm_strips(a.M, a.N);
    p.part = wg && !strips ? (float*)a.ws : nullptr;
    p.dw = a.dw;
    p.db = a.db;
    const bool sweeps = a.N > LONG_N || (a.N > FITS_N && (p.relu || p.drop.thr));
    const int64_t G = sweeps ? std::min<int64_t>(a.M, LONG_PARTS) : norm_parts(a.M, a.N);
    // dx over dy or x: not beside strips that read them
    auto clear = [&](const void* q, int64_t ld) {
        const int64_t es = a.dtype == MMVAE_T_F32 ? 4 : 2;
        const uintptr_t o = (uintptr_t)a.dx, i = (uintptr_t)q;
        return o + ((a.M - 1) * a.lddx + a.N) * es <= i || i + ((a.M - 1) * ld + a.N) * es <= o;
    };
    const bool apart = !a.dx || a.M < 1 || (clear(a.x, a.ldx) && clear(a.dy, a.lddy));
    auto go = [&](auto t, auto v, auto b) -> hipError_t {
        return by_flags(p, [&](auto m, auto e) {
            if constexpr (m.value && t.value * v.value * 8 > FITS_N) return hipErrorInvalidValue;  // (sweeps)
            else {
                const size_t lds = LnKeep<T, v.value, b.value, m.value, e.value>::B_HOLD ? 0 : (size_t)p.Np * 4;
                constexpr int RPB = b.value / t.value;
                const int64_t rows = strips ? (a.dx ? (a.M + RPB - 1) / RPB : 0) : G;
                const auto k = k_ln_bwd<T, t.value, v.value, b.value, m.value, e.value>;
                if (p.strips && apart)
                    return launch_lds(lds, k, dim3((unsigned)(p.strips + rows)), dim3(b.value), st, p);
                if (p.strips) {
                    OPCHK(launch(k_ln_strips<T, m.value, e.value>, dim3((unsigned)p.strips), dim3(STRIP_BLK), st, p));
                    p.strips = 0;
                }
                return rows ? launch_lds(lds, k, dim3((unsigned)rows), dim3(b.value), st, p) : hipSuccess;
            }
        });
    };
    if (a.M > 0 && strips) {  // (first: dx may overwrite dy or x)
        p.strip_waves = a.N > STRIP_N ? 2 : STRIP_BLK / 64;
        const int64_t each = STRIP_BLK / 64 / p.strip_waves;
        p.strips = (int)((p.Np / 8 + 8 * each - 1) / (8 * each) * 8);
        if (!sweeps) return by_width_strips(p.N, go);
        OPCHK(by_flags(p, [&](auto m, auto e) { return launch(k_ln_strips<T, m.value, e.value>, dim3((unsigned)p.strips), dim3(STRIP_BLK), st, p); }));
        return a.dx ? launch(k_ln_bwd_long<T>, dim3((unsigned)a.M), dim3(1024), st, p) : hipSuccess;
    }
    if (a.M > 0 && (a.dx || wg)) {
        if (sweeps) {
            if (wg)  // (first: dx may overwrite dy or x)
                OPCHK(launch(k_ln_cols<T>, dim3((unsigned)((p.Np / 8 + 255) / 256), (unsigned)G), dim3(256), st, p));
            if (a.dx) OPCHK(launch(k_ln_bwd_long<T>, dim3((unsigned)std::min<int64_t>(a.M, 512)), dim3(1024), st, p));
        } else {
            OPCHK(by_width_bwd(p.N, go));
        }
    }
    if (!wg) return hipSuccess;
    const dim3 grid((unsigned)((2 * p.Np + 31) / 32));
    const int parts = (int)(a.M > 0 ? G : 0);
    if (p.wf32)
        return launch(k_ln_wred<float>, grid, dim3(1024), st, p.N, p.Np, parts, (const float*)a.ws, (float*)a.dw, (float*)a.db);
    return launch(k_ln_wred<T>, grid, dim3(1024), st, p.N, p.Np, parts, (const float*)a.ws, (T*)a.dw, (T*)a.db);
}

}  // namespace mmvae
