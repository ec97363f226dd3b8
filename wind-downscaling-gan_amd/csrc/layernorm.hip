// layernorm.hip — LayerNormalization over the last axis of [P][C] tensors of any width, in fp32, bf16 or fp16, with unit channel
// stride and any row stride, and its backward pass with the reduction of the two parameter gradients.
//
//   forward   mean = sum_c x / C, var = sum_c (x - mean)^2 / C, rstd = 1 / sqrt(var + eps), z = (x - mean) rstd gamma + beta
//   backward  xh = (x - mean) rstd, a = dz gamma:  dx = rstd (a - mean_c a - xh mean_c(a xh)),
//             dgamma (+)= sum_rows dz xh,  dbeta (+)= sum_rows dz
//
// The norms of the networks (norms.hip: fp32 maps of at most 1024 channels, LeakyReLU derivative fused, parameter gradients through
// float atomics) stay what they are; these are for everything those refuse, and their parameter gradients are sums in a fixed order:
// the same bits on every run.
//
// Numerics: statistics, sums and the normalised value are fp32 whatever the tensors' type; z and dx are rounded once, on store.  The
// mean is corrected by the mean of (x - mean), which is what fp32 left out of it, so a row with an offset of many standard deviations
// keeps its digits; the variance is the sum of squares about the corrected mean.
//
// Bound: HBM where the tensors are larger than the caches — forward 2, backward 3 times the tensor, which is what the counters show.
// 16384 x 4096 bf16 forward 48.7 us (5.5 TB/s), backward 76 (5.3, the parameter sums' launch included); 65536 x 1024 fp32 90 and 135 us
// (5.9 and 6.0 TB/s); 2097152 x 16 fp32 backward 75 us (5.6, of which mean and rstd are 0.2).  A large copy reaches 5.3 TB/s on the same
// card.
#include "vec.h"
#include <algorithm>

// parameter c of gamma / beta: fp32 (ptype 0) or the 16-bit type of the activations; a missing vector reads as `none`
template <class T>
__device__ __forceinline__ float wdg_ln_param(const void* p, int ptype, int64_t c, float none) {
    if (!p) return none;
    return ptype == 0 ? static_cast<const float*>(p)[c] : (float)static_cast<const T*>(p)[c];
}

// ... V adjacent parameters in one or two requests
template <class T, int V>
__device__ __forceinline__ void wdg_ln_params(float (&r)[V], const void* p, int ptype, int64_t c, float none) {
    if (!p) {
#pragma unroll
        for (int j = 0; j < V; ++j) r[j] = none;
    } else if (ptype == 0) {
        const WdgVec<float, V> v = wdg_vec_load<float, V>(static_cast<const float*>(p) + c);
#pragma unroll
        for (int j = 0; j < V; ++j) r[j] = v.e[j];
    } else {
        const WdgVec<T, V> v = wdg_vec_load<T, V>(static_cast<const T*>(p) + c);
#pragma unroll
        for (int j = 0; j < V; ++j) r[j] = (float)v.e[j];
    }
}

// sum over the block's threads, result in every thread; `red` holds one float per wave, and may be reused after the next barrier
template <int NT>
__device__ __forceinline__ float wdg_ln_block_sum(float v, float* red) {
    v = wdg_wave_sum_fast(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) s += red[w];
    __syncthreads();
    return s;
}

// ---- rows that fit the registers of L lanes (C <= 16384) ------------------------------------------------------------------------
// L lanes (1 .. 64, a power of two; L == 0: all waves of the workgroup) hold a row, K vectors of V elements each, so x and dz are read once.  A thread's
// columns are the same for every row it meets: gamma, beta and the parameter sums stay in its registers while the workgroup walks
// over the rows.
//
// The last lanes of a row whose width is not L K V take the row's last V columns again instead of a shorter vector: their first `dup`
// elements belong to other lanes and count nowhere, what they store there is what the owner stores.  So every request is a whole
// vector inside the row, whatever the width.
template <int V, int K>
struct WdgLnCols {
    int col[K], dup[K];                                  // first column of vector k; elements j < dup are another lane's
    __device__ __forceinline__ WdgLnCols(int lanes, int sub, int C) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c0 = (k * lanes + sub) * V;
            col[k] = min(c0, C - V);
            dup[k] = c0 - col[k];
        }
    }
};

// U values summed over the lanes of each row, results in every lane.  A row of the whole workgroup goes through LDS, [U][16] floats at
// `red`, one barrier.  The caller gives two calls in a row different places: a wave that is ahead writes the second call's values while
// another one may still read the first's, and has passed the second's barrier, which that one reaches after reading, before the third.
template <int L, int U>
__device__ __forceinline__ void wdg_ln_row_sums(float (&v)[U], float* red) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if constexpr (L == 0 || L == 64) v[u] = wdg_wave_sum_fast(v[u]);
        else {
            if constexpr (L >= 2) v[u] = WDG_DPP_ADD(v[u], 0xB1);
            if constexpr (L >= 4) v[u] = WDG_DPP_ADD(v[u], 0x4E);
            if constexpr (L >= 8) v[u] = WDG_DPP_ADD(v[u], 0x141);
            if constexpr (L >= 16) v[u] = WDG_DPP_ADD(v[u], 0x140);
            if constexpr (L >= 32) v[u] += __shfl_xor(v[u], 16, 64);
        }
    }
    if constexpr (L == 0) {
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int u = 0; u < U; ++u) red[u * 16 + (threadIdx.x >> 6)] = v[u];
        }
        __syncthreads();
        // every lane takes one wave's value (lanes 0 .. 15 of each row of 16), the row sum adds them
        const int w = threadIdx.x & 15, waves = blockDim.x >> 6;
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = wdg_row16_sum(w < waves ? red[u * 16 + w] : 0.f);
    }
}

template <class T, int V, int K, int L, int NT, int U, bool TAIL, bool STREAM>
__global__ void __launch_bounds__(NT) wdg_layernorm_fwd_kernel(const T* x, int64_t ldx, const void* __restrict__ gamma,
                                                               const void* __restrict__ beta, int ptype, float eps, T* z, int64_t ldz,
                                                               float* mean_rstd, int64_t P, int C) {
    constexpr int RG = L ? NT / (L ? L : 1) : 1;         // rows at a time
    __shared__ float red[L ? 1 : 3 * U * 16];
    const int lanes = L ? L : blockDim.x, sub = threadIdx.x % lanes, g = threadIdx.x / lanes;
    const WdgLnCols<V, K> at(lanes, sub, C);
    const float invC = 1.f / (float)C;
    float gm[K][V], bt[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        wdg_ln_params<T, V>(gm[k], gamma, ptype, at.col[k], 1.f);
        wdg_ln_params<T, V>(bt[k], beta, ptype, at.col[k], 0.f);
    }
    const int64_t stride = (int64_t)gridDim.x * (RG * U);
    WdgVec<T, V> ahead[U][K];                            // the next rows are on their way while these are summed (behind the last: again the last)
    auto fetch = [&](int64_t p0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t p = std::min<int64_t>(p0 + u * RG + g, P - 1);
#pragma unroll
            for (int k = 0; k < K; ++k) ahead[u][k] = wdg_vec_load<T, V, STREAM>(x + p * ldx + at.col[k]);
        }
    };
    fetch((int64_t)blockIdx.x * (RG * U));
    for (int64_t p0 = (int64_t)blockIdx.x * (RG * U); p0 < P; p0 += stride) {
        WdgVec<T, V> xv[U][K];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < K; ++k) xv[u][k] = ahead[u][k];
        fetch(p0 + stride);
        float s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) s[u] += TAIL && j < at.dup[k] ? 0.f : (float)xv[u][k].e[j];
        }
        wdg_ln_row_sums<L, U>(s, red);
        float d2[2 * U];                                 // sums of (x - mean) and of its square
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] *= invC;
            d2[2 * u] = d2[2 * u + 1] = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float d = TAIL && j < at.dup[k] ? 0.f : (float)xv[u][k].e[j] - s[u];
                    d2[2 * u] += d;
                    d2[2 * u + 1] = fmaf(d, d, d2[2 * u + 1]);
                }
        }
        wdg_ln_row_sums<L, 2 * U>(d2, red + (L ? 0 : U * 16));
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t p = p0 + u * RG + g;
            const float corr = d2[2 * u] * invC;
            float var = fmaf(-corr, corr, d2[2 * u + 1] * invC);
            var = var < 0.f ? 0.f : var;                 // (a NaN stays one)
            const float rstd = 1.f / sqrtf(var + eps), shift = -corr * rstd;
            if (p < P) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    WdgVec<T, V> r;
#pragma unroll
                    for (int j = 0; j < V; ++j) r.e[j] = (T)fmaf(fmaf((float)xv[u][k].e[j] - s[u], rstd, shift), gm[k][j], bt[k][j]);
                    if (!TAIL || at.dup[k] < V) wdg_vec_store<T, V, STREAM>(z + p * ldz + at.col[k], r);
                }
                if (mean_rstd && sub == 0) {
                    mean_rstd[2 * p] = s[u] + corr;
                    mean_rstd[2 * p + 1] = rstd;
                }
            }
        }
    }
}

// part: NULL, or one row [dgamma | dbeta] (each of C rounded up to 4) of partial sums per workgroup
template <class T>
struct WdgLnBwd {
    const T* dz;
    int64_t lddz;
    const T* x;
    int64_t ldx;
    const float* mean_rstd;
    const void* gamma;
    int ptype;
    T* dx;
    int64_t lddx, P;
    int C;
};
// the rows of workgroup `blk` of `nblk`
template <class T, int V, int K, int L, int NT, int U, bool TAIL, bool STREAM>
__device__ __forceinline__ void wdg_ln_bwd_rows(const WdgLnBwd<T>& q, float* part, int blk, int nblk) {
    const T *dz = q.dz, *x = q.x;
    T* dx = q.dx;
    const float* __restrict__ mean_rstd = q.mean_rstd;
    const int64_t lddz = q.lddz, ldx = q.ldx, lddx = q.lddx, P = q.P;
    const int C = q.C;
    constexpr int RG = L ? NT / (L ? L : 1) : 1, COPIES = L ? NT / 64 : 1;      // waves that hold sums of the same columns
    constexpr bool AHEAD = K * U <= 2 && NT <= 512;
    __shared__ float red[L ? 1 : 2 * 2 * U * 16];
    __shared__ float gather[COPIES > 1 ? NT * V : 1];
    const int lanes = L ? L : blockDim.x, t = threadIdx.x, sub = t % lanes, g = t / lanes;
    const WdgLnCols<V, K> at(lanes, sub, C);
    const float invC = 1.f / (float)C;
    float gm[K][V], sg[K][V], sb[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        wdg_ln_params<T, V>(gm[k], q.gamma, q.ptype, at.col[k], 1.f);
#pragma unroll
        for (int j = 0; j < V; ++j) sg[k][j] = sb[k][j] = 0.f;
    }
    int turn = 0;
    const int64_t stride = (int64_t)nblk * (RG * U);
    WdgVec<T, V> x_a[U][K], g_a[U][K];                   // the next rows, on their way while these are worked on (behind the last: again the last)
    float mean_a[U], rstd_a[U];
    auto fetch = [&](int64_t p0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t p = std::min<int64_t>(p0 + u * RG + g, P - 1);
            mean_a[u] = mean_rstd[2 * p];
            rstd_a[u] = mean_rstd[2 * p + 1];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                x_a[u][k] = wdg_vec_load<T, V, STREAM>(x + p * ldx + at.col[k]);
                g_a[u][k] = wdg_vec_load<T, V, STREAM>(dz + p * lddz + at.col[k]);
            }
        }
    };
    if constexpr (AHEAD) fetch((int64_t)blk * (RG * U));
    for (int64_t p0 = (int64_t)blk * (RG * U); p0 < P; p0 += stride) {
        WdgVec<T, V> xv[U][K], gv[U][K];
        float mean[U], rstd[U], s[2 * U];
        if constexpr (!AHEAD) fetch(p0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            mean[u] = mean_a[u];
            rstd[u] = rstd_a[u];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                xv[u][k] = x_a[u][k];
                gv[u][k] = g_a[u][k];
            }
        }
        if constexpr (AHEAD) fetch(p0 + stride);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool on = p0 + u * RG + g < P;
            s[2 * u] = s[2 * u + 1] = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    // (every multiply-add is written as one: the instances then give the same bits)
                    const float gg = (float)gv[u][k].e[j], xh = ((float)xv[u][k].e[j] - mean[u]) * rstd[u], a = gg * gm[k][j];
                    const float n0 = fmaf(gg, gm[k][j], s[2 * u]), n1 = fmaf(a, xh, s[2 * u + 1]);
                    s[2 * u] = TAIL && j < at.dup[k] ? s[2 * u] : n0;
                    s[2 * u + 1] = TAIL && j < at.dup[k] ? s[2 * u + 1] : n1;
                    if (on) {                            // (elements j < dup gather too, and are left out below)
                        sg[k][j] = fmaf(gg, xh, sg[k][j]);
                        sb[k][j] += gg;
                    }
                }
        }
        wdg_ln_row_sums<L, 2 * U>(s, red + (L ? 0 : turn * 2 * U * 16));
        turn ^= 1;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t p = p0 + u * RG + g;
            const float m1 = s[2 * u] * invC, m2 = s[2 * u + 1] * invC;
            if (p < P) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    WdgVec<T, V> r;
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float xh = ((float)xv[u][k].e[j] - mean[u]) * rstd[u];
                        r.e[j] = (T)(rstd[u] * fmaf(-xh, m2, fmaf((float)gv[u][k].e[j], gm[k][j], -m1)));
                    }
                    if (!TAIL || at.dup[k] < V) wdg_vec_store<T, V, STREAM>(dx + p * lddx + at.col[k], r);
                }
            }
        }
    }
    if (!part) return;
    // the workgroup's sums of each column, in a fixed order: lanes of a wave that hold the same columns, then the holders through LDS
    const int Cp = (C + 3) & ~3;
    float* row = part + (int64_t)blk * 2 * Cp;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            float v[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[j] = which ? sb[k][j] : sg[k][j];
#pragma unroll
                for (int o = L ? L : 64; o < 64; o <<= 1) v[j] += __shfl_xor(v[j], o, 64);
            }
            if constexpr (COPIES > 1) {
                __syncthreads();
#pragma unroll
                for (int j = 0; j < V; ++j) gather[j * NT + t] = v[j];
                __syncthreads();
                if (t < lanes) {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        v[j] = 0.f;
#pragma unroll
                        for (int w = 0; w < COPIES; ++w) v[j] += gather[j * NT + w * 64 + t];
                    }
                }
            }
            if (t < lanes) {
                if (!TAIL || at.dup[k] == 0) {
                    WdgVec<float, V> r;
#pragma unroll
                    for (int j = 0; j < V; ++j) r.e[j] = v[j];
                    wdg_vec_store<float, V>(row + which * Cp + at.col[k], r);
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if (j >= at.dup[k]) row[which * Cp + at.col[k] + j] = v[j];
                }
            }
        }
}

template <class T, int V, int K, int L, int NT, int U, bool TAIL, bool STREAM>
__global__ void __launch_bounds__(NT) wdg_layernorm_bwd_kernel(const WdgLnBwd<T> q, float* part) {
    wdg_ln_bwd_rows<T, V, K, L, NT, U, TAIL, STREAM>(q, part, blockIdx.x, gridDim.x);
}

// Few rows, dx apart from x and dz: both parameter gradients in the same launch, by workgroups of their own behind the `rowblocks` that
// form dx.  Each owns `cols` columns and reads them of all rows again — from the cache, there are few —, blockDim / cols rows at a time,
// added in that order and then over the threads.  No partial sums, no second launch.
constexpr int LN_FEW_ROWS = 512;
template <class T, int V, int K, int L, int NT, int U>
__global__ void __launch_bounds__(NT) wdg_layernorm_bwd_few_kernel(const WdgLnBwd<T> q, int rowblocks, int cols, float* dgamma, float* dbeta, int accumulate) {
    if ((int)blockIdx.x < rowblocks) {
        wdg_ln_bwd_rows<T, V, K, L, NT, U, true, false>(q, nullptr, blockIdx.x, rowblocks);
        return;
    }
    __shared__ float sums[2][NT];
    const int t = threadIdx.x, c0 = ((int)blockIdx.x - rowblocks) * cols, c = c0 + t % cols, sets = blockDim.x / cols;
    float sg = 0.f, sb = 0.f;
    if (c < q.C) {
#pragma unroll 8
        for (int64_t p = t / cols; p < q.P; p += sets) {
            const float g = (float)q.dz[p * q.lddz + c], xh = ((float)q.x[p * q.ldx + c] - q.mean_rstd[2 * p]) * q.mean_rstd[2 * p + 1];
            sg = fmaf(g, xh, sg);
            sb += g;
        }
    }
    sums[0][t] = sg;
    sums[1][t] = sb;
    __syncthreads();
    if (t < 2 * cols) {
        const int which = t / cols, cc = c0 + t % cols;
        float s = 0.f;
        for (int w = 0; w < sets; ++w) s += sums[which][w * cols + t % cols];
        float* dst = which ? dbeta : dgamma;
        if (dst && cc < q.C) dst[cc] = (accumulate ? dst[cc] : 0.f) + s;
    }
}

// ---- any width: one block per row, the row read once per pass (from the cache, but for the first) -------------------------------------
// 4096 x 32768 bf16: forward 181 us (3.0 TB/s, each tensor counted once), backward 326 (2.5).
// The last, partial vector of a row is taken element by element (never beyond the row: what follows may be another row, or nothing).
constexpr int LNW_NT = 1024;

template <class T, int V, class F>
__device__ __forceinline__ void wdg_ln_row(const T* x, int64_t C, F&& f) {
    for (int64_t c = (int64_t)threadIdx.x * V; c < C; c += (int64_t)LNW_NT * V) {
        if (c + V <= C) {
            const WdgVec<T, V> v = wdg_vec_load<T, V>(x + c);
            f(c, V, v);
        } else {
            WdgVec<T, V> v;
            const int n = (int)(C - c);
#pragma unroll
            for (int j = 0; j < V; ++j) v.e[j] = j < n ? x[c + j] : (T)0.f;
            f(c, n, v);
        }
    }
}
// the parameters beside n elements from column c on
template <class T, int V>
__device__ __forceinline__ void wdg_ln_params_of(float (&r)[V], const void* p, int ptype, int64_t c, int n, float none) {
    if (n == V) wdg_ln_params<T, V>(r, p, ptype, c, none);
    else
#pragma unroll
        for (int j = 0; j < V; ++j) r[j] = wdg_ln_param<T>(p, ptype, j < n ? c + j : c, none);
}
template <class T, int V>
__device__ __forceinline__ void wdg_ln_put(T* p, int n, const WdgVec<T, V>& v) {
    if (n == V) wdg_vec_store<T, V>(p, v);
    else
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < n) p[j] = v.e[j];
}

template <class T, int V>
__global__ void __launch_bounds__(LNW_NT) wdg_layernorm_fwd_wide_kernel(const T* x, int64_t ldx, const void* __restrict__ gamma,
                                                                        const void* __restrict__ beta, int ptype, float eps, T* z,
                                                                        int64_t ldz, float* mean_rstd, int64_t P, int64_t C) {
    __shared__ float red[LNW_NT / 64];
    const float invC = 1.f / (float)C;
    for (int64_t p = blockIdx.x; p < P; p += gridDim.x) {
        const T* xr = x + p * ldx;
        T* zr = z + p * ldz;
        float s = 0.f;
        wdg_ln_row<T, V>(xr, C, [&](int64_t, int n, const WdgVec<T, V>& v) {
#pragma unroll
            for (int j = 0; j < V; ++j) s += j < n ? (float)v.e[j] : 0.f;
        });
        const float mean0 = wdg_ln_block_sum<LNW_NT>(s, red) * invC;
        float e = 0.f, q = 0.f;
        wdg_ln_row<T, V>(xr, C, [&](int64_t, int n, const WdgVec<T, V>& v) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = j < n ? (float)v.e[j] - mean0 : 0.f;
                e += d;
                q += d * d;
            }
        });
        const float corr = wdg_ln_block_sum<LNW_NT>(e, red) * invC;
        float var = wdg_ln_block_sum<LNW_NT>(q, red) * invC - corr * corr;
        var = var < 0.f ? 0.f : var;                       // (a NaN stays one)
        const float rstd = 1.f / sqrtf(var + eps);
        wdg_ln_row<T, V>(xr, C, [&](int64_t c, int n, const WdgVec<T, V>& v) {
            WdgVec<T, V> r;
            float gm[V], bt[V];
            wdg_ln_params_of<T, V>(gm, gamma, ptype, c, n, 1.f);
            wdg_ln_params_of<T, V>(bt, beta, ptype, c, n, 0.f);
#pragma unroll
            for (int j = 0; j < V; ++j) r.e[j] = (T)((((float)v.e[j] - mean0) - corr) * rstd * gm[j] + bt[j]);
            wdg_ln_put<T, V>(zr + c, n, r);
        });
        if (mean_rstd && threadIdx.x == 0) {
            mean_rstd[2 * p] = mean0 + corr;
            mean_rstd[2 * p + 1] = rstd;
        }
    }
}

// dx alone (the parameter sums read x and dz in a launch of their own, before: dx may be written over either)
template <class T, int V>
__global__ void __launch_bounds__(LNW_NT) wdg_layernorm_bwd_wide_kernel(const T* dz, int64_t lddz, const T* x, int64_t ldx,
                                                                        const float* __restrict__ mean_rstd, const void* __restrict__ gamma,
                                                                        int ptype, T* dx, int64_t lddx, int64_t P, int64_t C) {
    __shared__ float red[LNW_NT / 64];
    const float invC = 1.f / (float)C;
    for (int64_t p = blockIdx.x; p < P; p += gridDim.x) {
        const float mean = mean_rstd[2 * p], rstd = mean_rstd[2 * p + 1];
        const T* xr = x + p * ldx;
        const T* gr = dz + p * lddz;
        T* dr = dx + p * lddx;
        float s1 = 0.f, s2 = 0.f;
        auto other = [&](int64_t c, int n) {               // x beside dz, of the same n elements
            WdgVec<T, V> u;
            if (n == V) return wdg_vec_load<T, V>(xr + c);
#pragma unroll
            for (int j = 0; j < V; ++j) u.e[j] = j < n ? xr[c + j] : (T)0.f;
            return u;
        };
        wdg_ln_row<T, V>(gr, C, [&](int64_t c, int n, const WdgVec<T, V>& g) {
            const WdgVec<T, V> u = other(c, n);
            float gm[V];
            wdg_ln_params_of<T, V>(gm, gamma, ptype, c, n, 1.f);
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j < n) {
                    const float a = (float)g.e[j] * gm[j];
                    s1 += a;
                    s2 += a * (((float)u.e[j] - mean) * rstd);
                }
        });
        s1 = wdg_ln_block_sum<LNW_NT>(s1, red) * invC;
        s2 = wdg_ln_block_sum<LNW_NT>(s2, red) * invC;
        wdg_ln_row<T, V>(gr, C, [&](int64_t c, int n, const WdgVec<T, V>& g) {
            const WdgVec<T, V> u = other(c, n);
            WdgVec<T, V> r;
            float gm[V];
            wdg_ln_params_of<T, V>(gm, gamma, ptype, c, n, 1.f);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float a = (float)g.e[j] * gm[j];
                r.e[j] = (T)(rstd * (a - s1 - ((float)u.e[j] - mean) * rstd * s2));
            }
            wdg_ln_put<T, V>(dr + c, n, r);
        });
    }
}

// ---- parameter gradients -----------------------------------------------------------------------------------------------------------
// Partial sums [slice][dgamma | dbeta][C, rounded up to 4]: a block owns 256 V columns of one slice of the rows (C >= V; the last vector
// reaches back over columns of its neighbour, whose sums it does not store).
template <class T, int V>
__global__ void __launch_bounds__(256) wdg_layernorm_colsum_kernel(const T* __restrict__ dz, int64_t lddz, const T* __restrict__ x,
                                                                   int64_t ldx, const float* __restrict__ mean_rstd, float* part,
                                                                   int64_t P, int64_t C, int slices) {
    const int64_t c0 = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
    if (c0 >= C) return;
    const int64_t c = std::min<int64_t>(c0, C - V);
    const int64_t per = (P + slices - 1) / slices, p0 = blockIdx.y * per, p1 = std::min<int64_t>(P, p0 + per);
    float sg[V], sb[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sg[j] = sb[j] = 0.f;
    constexpr int U = 4;
    for (int64_t p = p0; p < p1; p += U) {
        WdgVec<T, V> xv[U], gv[U];
        float mean[U], rstd[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t q = std::min<int64_t>(p + u, P - 1);
            mean[u] = mean_rstd[2 * q];
            rstd[u] = mean_rstd[2 * q + 1];
            xv[u] = wdg_vec_load<T, V>(x + q * ldx + c);
            gv[u] = wdg_vec_load<T, V>(dz + q * lddz + c);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (p + u >= p1) break;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float g = (float)gv[u].e[j];
                sg[j] += g * (((float)xv[u].e[j] - mean[u]) * rstd[u]);
                sb[j] += g;
            }
        }
    }
    const int64_t Cp = (C + 3) & ~3ll;
    float* row = part + (int64_t)blockIdx.y * 2 * Cp;
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (c + j >= c0) {
            row[c + j] = sg[j];
            row[Cp + c + j] = sb[j];
        }
}

// dgamma / dbeta (+)= the sum of the partial rows, in the rows' order within each of the 1024 / CB interleaved sets and then over the
// sets as a tree: a block owns CB of the 2 C columns
template <int CB>
__global__ void __launch_bounds__(1024) wdg_layernorm_finish_kernel(const float* __restrict__ part, int rows, int64_t C, float* dgamma,
                                                                    float* dbeta, int accumulate) {
    constexpr int SETS = 1024 / CB;
    __shared__ float red[1024];
    const int t = threadIdx.x;
    const int64_t col = (int64_t)blockIdx.x * CB + t % CB, Cp = (C + 3) & ~3ll;
    float s = 0.f;
    if (col < 2 * Cp) {
#pragma unroll 8
        for (int r = t / CB; r < rows; r += SETS) s += part[(int64_t)r * 2 * Cp + col];
    }
    red[t] = s;
    __syncthreads();
    for (int o = SETS / 2; o > 0; o >>= 1) {
        if (t < o * CB) red[t] += red[t + o * CB];
        __syncthreads();
    }
    if (t < CB && col < 2 * Cp) {
        float* dst = col < Cp ? dgamma : dbeta;
        const int64_t c = col < Cp ? col : col - Cp;
        if (dst && c < C) dst[c] = (accumulate ? dst[c] : 0.f) + red[t];
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------------------------
// How a [P][C] tensor is cut: elements per vector, lanes per row (0: a workgroup of NT threads), vectors per lane, rows in flight per
// thread.  K == 0: the row does not fit (the kernels that read it once per pass take it).
struct LnGeom {
    int V, L, K, NT, U;
    int blocks;                                          // of the register kernels; rows of the backward's table of partial sums
};
constexpr int LN_CUS = 256;
constexpr int64_t LN_MAX_ROW = 16384;                    // widest row that a workgroup holds in registers

static LnGeom ln_geom(int64_t P, int64_t C, int type, bool bwd) {
    LnGeom g = {type == WDG_F32 ? 4 : 8, 0, 0, 256, 1, 0};
    if (C < g.V) {
        g.V = 1;
        g.L = 8;
        g.K = 1;
        g.U = 4;
    } else {
        const int64_t vecs = (C + g.V - 1) / g.V;
        const int wave = g.V == 4 ? 4 : 2;               // vectors per lane of a row that one wave holds: at most 16 elements
        if (vecs <= 64) {
            g.L = 1;
            while (g.L < vecs) g.L <<= 1;
            g.K = 1;
            g.U = 4;
        } else if (vecs <= 64 * wave) {
            g.L = 64;
            g.K = vecs <= 128 ? 2 : 4;
            g.U = 4 / g.K;
        } else if (C <= LN_MAX_ROW) {
            g.K = wave;
            g.NT = (int)((vecs + 64 * g.K - 1) / (64 * g.K)) * 64;
            // Forward, 16-bit types: two rows per barrier, except in workgroups of 5 to 8 waves (us with one / two rows: 16384 x 4096
            // 54.4 / 50.5, 16384 x 10000 157 / 131, but 16384 x 8192 97 / 104 and 16384 x 5003 68 / 74).  With 32-bit elements twice
            // the bytes per row are on their way already: 16384 x 4096 97 / 101, 4096 x 16384 97 / 115.
            g.U = !bwd && g.V == 8 && (g.NT <= 256 || g.NT > 512) ? 2 : 1;
        }
    }
    if (g.K) {
        // Threads per compute unit: a workgroup that stays walks over many rows with its parameters in registers, and each one of the
        // backward writes 8 C bytes of partial sums, so no more of them than keep the memory busy.  Backward, us with 512 / 1024:
        // 16384 x 4096 bf16 81 / 94, 32768 x 2048 bf16 81 / 95, 262144 x 256 fp32 151 / 156.  (The quotient is cut to a whole number: a
        // backward workgroup of 320 to 448 threads has its compute unit to itself.)  Forward, us with 1024 / 2048: 16384 x 4097
        // bf16 (320 threads) 65 / 78, 16384 x 5003 fp16 68 / 75; 4194304 x 16 bf16 57 / 57, 32768 x 2048 bf16 51 / 51.
        const int threads = bwd ? 512 : g.NT > 256 ? 1024 : 2048;
        const int64_t rows = (int64_t)(g.L ? g.NT / g.L : 1) * g.U, resident = LN_CUS * std::max(1, threads / g.NT);
        // (backward: three rows at least for a row of partial sums; 768 x 4096 bf16 17.7 -> 13.1 us)
        const int64_t least = rows * (bwd && !g.L ? 3 : 1);
        g.blocks = (int)std::max<int64_t>(1, std::min<int64_t>((P + least - 1) / least, resident));
    } else {
        const int64_t tiles = (C + 256 * g.V - 1) / (256 * g.V);
        g.blocks = (int)std::max<int64_t>(1, std::min<int64_t>((P + 15) / 16, std::max<int64_t>(1, 1024 / tiles)));
    }
    return g;
}

// f.template run<V, K, L, NT, U>() for the geometry, NT the most threads the instance is built for; false: no register kernel for it
template <int V, int U, class F>
static void ln_dispatch_block(const LnGeom& g, F& f) {
    constexpr int K = V == 4 ? 4 : 2;
    if (g.NT <= 256) f.template run<V, K, 0, 256, U>();
    else if (g.NT <= 512) f.template run<V, K, 0, 512, 1>();
    else f.template run<V, K, 0, 1024, U>();
}
template <int V, class F>
static bool ln_dispatch(const LnGeom& g, F& f) {
    if (g.K == 0) return false;
    if (g.V == 1) {
        f.template run<1, 1, 8, 256, 4>();
        return true;
    }
    switch (g.L) {
        case 1: f.template run<V, 1, 1, 256, 4>(); break;
        case 2: f.template run<V, 1, 2, 256, 4>(); break;
        case 4: f.template run<V, 1, 4, 256, 4>(); break;
        case 8: f.template run<V, 1, 8, 256, 4>(); break;
        case 16: f.template run<V, 1, 16, 256, 4>(); break;
        case 32: f.template run<V, 1, 32, 256, 4>(); break;
        case 64:
            if (g.K == 1) f.template run<V, 1, 64, 256, 4>();
            else if (g.K == 2) f.template run<V, 2, 64, 256, 2>();
            else if constexpr (V == 4) f.template run<V, 4, 64, 256, 1>();
            break;
        default: ln_dispatch_block<V, V == 8 ? F::BLOCK_U16 : 1>(g, f);
    }
    return true;
}

// Tensors that together pass the chip's last-level cache (256 MiB) are streamed past it.  us without / with: 16384 x 4096 fp32 forward
// 97 / 92, backward 153 / 138; 16384 x 8192 bf16 97 / 89, 154 / 142; 65536 x 1024 bf16 backward 80 / 73.  Below that size the tensors may
// still be there from the launch before, and stay for the one behind (512 x 4096 bf16 9.4 / 9.9); rows that are not whole vectors of all
// lanes gain nothing (16384 x 10000 bf16 backward 207 / 210).
static bool ln_stream(int64_t bytes) { return bytes >= 256ll << 20; }

static bool ln_types_ok(int type, int ptype) {
    return type >= WDG_F32 && type <= WDG_F16 && (ptype == WDG_F32 || ptype == type);
}
static bool ln_aligned(const void* p, int type) { return ((uintptr_t)p & (type == WDG_F32 ? 3 : 1)) == 0; }
static const int64_t LN_MAX_C = 1ll << 24;      // (C itself is exact in fp32)

template <class T>
struct LnFwd {
    static constexpr int BLOCK_U16 = 2;
    const T* x;
    int64_t ldx;
    const void *gamma, *beta;
    int ptype;
    float eps;
    T* z;
    int64_t ldz;
    float* mean_rstd;
    int64_t P, C;
    hipStream_t st;
    LnGeom g;
    template <int V, int K, int L, int NT, int U>
    void run() {
        const bool whole = C == (int64_t)V * K * (L ? L : g.NT);
        const auto kernel = !whole ? wdg_layernorm_fwd_kernel<T, V, K, L, NT, U, true, false>
                            : ln_stream(2 * P * C * sizeof(T)) ? wdg_layernorm_fwd_kernel<T, V, K, L, NT, U, false, true>
                                                                : wdg_layernorm_fwd_kernel<T, V, K, L, NT, U, false, false>;
        hipLaunchKernelGGL(kernel, dim3(g.blocks), dim3(g.NT), 0, st, x, ldx, gamma, beta, ptype, eps, z, ldz, mean_rstd, P, (int)C);
    }
};

template <class T, int V>
static int ln_fwd_launch(const void* x, int64_t ldx, const void* gamma, const void* beta, int ptype, float eps, void* z, int64_t ldz,
                         float* mean_rstd, int64_t P, int64_t C, int type, hipStream_t st) {
    LnFwd<T> f = {(const T*)x, ldx, gamma, beta, ptype, eps, (T*)z, ldz, mean_rstd, P, C, st, ln_geom(P, C, type, false)};
    if (!ln_dispatch<V>(f.g, f))
        hipLaunchKernelGGL((wdg_layernorm_fwd_wide_kernel<T, V>), dim3((unsigned)std::min<int64_t>(P, 4096)), dim3(LNW_NT), 0, st, (const T*)x, ldx,
                           gamma, beta, ptype, eps, (T*)z, ldz, mean_rstd, P, C);
    WDG_LAUNCH_CHECK();
    return WDG_OK;
}

extern "C" int wdg_layernorm_fwd(const void* x, int64_t ldx, const void* gamma, const void* beta, float eps, void* z, int64_t ldz,
                                 float* mean_rstd, int64_t P, int64_t C, int type, int param_type, wdg_stream stream) {
    WDG_CHECK_ARG(ln_types_ok(type, param_type), "type: fp32, bf16 or fp16; parameters: fp32 or that type");
    WDG_CHECK_ARG(P >= 0 && C >= 1 && C <= LN_MAX_C, "bad sizes");
    if (P == 0) return WDG_OK;
    WDG_CHECK_ARG(x && z, "null argument");
    WDG_CHECK_ARG(eps >= 0.f, "eps has to be a number, not negative");
    WDG_CHECK_ARG(ln_aligned(x, type) && ln_aligned(z, type) && ln_aligned(gamma, param_type) && ln_aligned(beta, param_type) && ln_aligned(mean_rstd, WDG_F32),
                  "not aligned to its element");
    WDG_CHECK_ARG(ldx >= 0 && (P == 1 || ldz >= C), "output rows overlap");
    hipStream_t st = (hipStream_t)stream;
    if (type == WDG_F32) return ln_fwd_launch<float, 4>(x, ldx, gamma, beta, param_type, eps, z, ldz, mean_rstd, P, C, type, st);
    if (type == WDG_BF16) return ln_fwd_launch<__bf16, 8>(x, ldx, gamma, beta, param_type, eps, z, ldz, mean_rstd, P, C, type, st);
    return ln_fwd_launch<_Float16, 8>(x, ldx, gamma, beta, param_type, eps, z, ldz, mean_rstd, P, C, type, st);
}

extern "C" size_t wdg_layernorm_bwd_ws_bytes(int64_t P, int64_t C, int type) {
    if (P <= 0 || C <= 0 || C > LN_MAX_C || type < WDG_F32 || type > WDG_F16) return 0;
    const LnGeom g = ln_geom(P, C, type, true);
    return (size_t)g.blocks * 2 * (size_t)((C + 3) & ~3ll) * sizeof(float);
}

static int ln_finish(const float* part, int rows, int64_t C, float* dgamma, float* dbeta, int accumulate, hipStream_t st) {
    const int64_t cols = 2 * ((C + 3) & ~3ll);
    // columns per workgroup by how many workgroups they leave: with 64 / 32, us of the whole backward: 3000 x 1024 bf16 12.1 / 10.8,
    // 1537 x 5003 fp16 18.4 / 19.5
    if (cols <= 256)
        hipLaunchKernelGGL(wdg_layernorm_finish_kernel<16>, dim3((unsigned)((cols + 15) / 16)), dim3(1024), 0, st, part, rows, C, dgamma, dbeta, accumulate);
    else if (cols <= 4096)
        hipLaunchKernelGGL(wdg_layernorm_finish_kernel<32>, dim3((unsigned)((cols + 31) / 32)), dim3(1024), 0, st, part, rows, C, dgamma, dbeta, accumulate);
    else
        hipLaunchKernelGGL(wdg_layernorm_finish_kernel<64>, dim3((unsigned)((cols + 63) / 64)), dim3(1024), 0, st, part, rows, C, dgamma, dbeta, accumulate);
    WDG_LAUNCH_CHECK();
    return WDG_OK;
}

template <class T>
struct LnBwd {
    static constexpr int BLOCK_U16 = 1;
    WdgLnBwd<T> q;
    float *part, *dgamma, *dbeta;
    int accumulate;
    bool few;                                            // wdg_layernorm_bwd_few_kernel
    hipStream_t st;
    LnGeom g;
    template <int V, int K, int L, int NT, int U>
    void run() {
        if (few) {
            // 16 columns per workgroup, more rows at a time, where that still gives few workgroups; us with 16 / 32 columns / in two launches:
            // 256 x 64 fp32 3.3 / 4.1 / 5.2, 512 x 1024 bf16 4.1 / 5.5 / 7.7, 512 x 4096 bf16 8.5 / 6.3 / 16, 256 x 16384 bf16 20 / 14 / 21;
            // with 1024 rows: 64 columns fp32 6.3 / 10 / 5.3 (where LN_FEW_ROWS ends; more rows of wide tensors were not measured in one launch)
            const int cols = q.C <= 2048 ? 16 : 32, colblocks = (q.C + cols - 1) / cols, rows = (L ? NT / (L ? L : 1) : 1) * U;
            const int rowblocks = (int)((q.P + rows - 1) / rows);
            hipLaunchKernelGGL((wdg_layernorm_bwd_few_kernel<T, V, K, L, NT, U>), dim3(rowblocks + colblocks), dim3(g.NT), 0, st, q, rowblocks, cols, dgamma, dbeta, accumulate);
            return;
        }
        const bool whole = q.C == (int64_t)V * K * (L ? L : g.NT);
        const auto kernel = !whole ? wdg_layernorm_bwd_kernel<T, V, K, L, NT, U, true, false>
                            : ln_stream(3 * q.P * q.C * sizeof(T)) ? wdg_layernorm_bwd_kernel<T, V, K, L, NT, U, false, true>
                                                                    : wdg_layernorm_bwd_kernel<T, V, K, L, NT, U, false, false>;
        hipLaunchKernelGGL(kernel, dim3(g.blocks), dim3(g.NT), 0, st, q, part);
    }
};

// whether the memory that the rows of two [P][C] tensors of `size` bytes per element span meets
static bool ln_meet(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t P, int64_t C, int size) {
    const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
    return a0 < b0 + (uintptr_t)(((P - 1) * ldb + C) * size) && b0 < a0 + (uintptr_t)(((P - 1) * lda + C) * size);
}

template <class T, int V>
static int ln_bwd_launch(const void* dz, int64_t lddz, const void* x, int64_t ldx, const float* mean_rstd, const void* gamma, int ptype,
                         void* dx, int64_t lddx, float* dgamma, float* dbeta, int accumulate, int64_t P, int64_t C, int type, float* part,
                         hipStream_t st) {
    const bool params = dgamma || dbeta;
    if (P == 0) return params ? ln_finish(part, 0, C, dgamma, dbeta, accumulate, st) : WDG_OK;
    const bool few = params && P <= LN_FEW_ROWS && C <= LN_MAX_ROW && !ln_meet(dx, lddx, x, ldx, P, C, sizeof(T)) && !ln_meet(dx, lddx, dz, lddz, P, C, sizeof(T));
    LnBwd<T> f = {{(const T*)dz, lddz, (const T*)x, ldx, mean_rstd, gamma, ptype, (T*)dx, lddx, P, (int)C}, params ? part : nullptr, dgamma, dbeta, accumulate,
                  few, st, ln_geom(P, C, type, true)};
    if (!ln_dispatch<V>(f.g, f)) {
        if (params) {
            hipLaunchKernelGGL((wdg_layernorm_colsum_kernel<T, V>), dim3((unsigned)((C + 256 * V - 1) / (256 * V)), f.g.blocks), dim3(256), 0, st,
                               (const T*)dz, lddz, (const T*)x, ldx, mean_rstd, part, P, C, f.g.blocks);
            WDG_LAUNCH_CHECK();
        }
        hipLaunchKernelGGL((wdg_layernorm_bwd_wide_kernel<T, V>), dim3((unsigned)std::min<int64_t>(P, 4096)), dim3(LNW_NT), 0, st, (const T*)dz,
                           lddz, (const T*)x, ldx, mean_rstd, gamma, ptype, (T*)dx, lddx, P, C);
    }
    WDG_LAUNCH_CHECK();
    return params && !few ? ln_finish(part, f.g.blocks, C, dgamma, dbeta, accumulate, st) : WDG_OK;
}

extern "C" int wdg_layernorm_bwd(const void* dz, int64_t lddz, const void* x, int64_t ldx, const float* mean_rstd, const void* gamma,
                                 void* dx, int64_t lddx, float* dgamma, float* dbeta, int accumulate, int64_t P, int64_t C, int type,
                                 int param_type, void* ws, size_t ws_bytes, wdg_stream stream) {
    WDG_CHECK_ARG(ln_types_ok(type, param_type), "type: fp32, bf16 or fp16; parameters: fp32 or that type");
    WDG_CHECK_ARG(P >= 0 && C >= 1 && C <= LN_MAX_C, "bad sizes");
    WDG_CHECK_ARG(P == 0 || (dz && x && mean_rstd && dx), "null argument");
    WDG_CHECK_ARG(lddz >= 0 && ldx >= 0 && (P <= 1 || lddx >= C), "gradient rows overlap");
    WDG_CHECK_ARG(ln_aligned(dz, type) && ln_aligned(x, type) && ln_aligned(dx, type) && ln_aligned(gamma, param_type) && ln_aligned(mean_rstd, WDG_F32) &&
                      ln_aligned(dgamma, WDG_F32) && ln_aligned(dbeta, WDG_F32) && ln_aligned(ws, WDG_F32), "not aligned to its element");
    if (P > 0 && (dgamma || dbeta) && (!ws || ws_bytes < wdg_layernorm_bwd_ws_bytes(P, C, type))) {
        wdg_set_error("wdg_layernorm_bwd: workspace too small");
        return WDG_ERR_WORKSPACE;
    }
    hipStream_t st = (hipStream_t)stream;
    float* part = (float*)ws;
    if (type == WDG_F32)
        return ln_bwd_launch<float, 4>(dz, lddz, x, ldx, mean_rstd, gamma, param_type, dx, lddx, dgamma, dbeta, accumulate, P, C, type, part, st);
    if (type == WDG_BF16)
        return ln_bwd_launch<__bf16, 8>(dz, lddz, x, ldx, mean_rstd, gamma, param_type, dx, lddx, dgamma, dbeta, accumulate, P, C, type, part, st);
    return ln_bwd_launch<_Float16, 8>(dz, lddz, x, ldx, mean_rstd, gamma, param_type, dx, lddx, dgamma, dbeta, accumulate, P, C, type, part, st);
}
