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
#include "vec.h"
#include <algorithm>

// parameter c of gamma / beta: fp32 (ptype 0) or the 16-bit type of the activations; a missing vector reads as `none`
template <class T>
__device__ __forceinline__ float wdg_ln_param(const void* p, int ptype, int64_t c, float none) {
    if (!p) return none;
    return ptype == 0 ? static_cast<const float*>(p)[c] : (float)static_cast<const T*>(p)[c];
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

// ---- any width: one block per row, the row read once per pass -------------------------------------------------------------------
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
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int64_t cc = j < n ? c + j : c;
                r.e[j] = (T)((((float)v.e[j] - mean0) - corr) * rstd * wdg_ln_param<T>(gamma, ptype, cc, 1.f) + wdg_ln_param<T>(beta, ptype, cc, 0.f));
            }
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
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j < n) {
                    const float a = (float)g.e[j] * wdg_ln_param<T>(gamma, ptype, c + j, 1.f);
                    s1 += a;
                    s2 += a * (((float)u.e[j] - mean) * rstd);
                }
        });
        s1 = wdg_ln_block_sum<LNW_NT>(s1, red) * invC;
        s2 = wdg_ln_block_sum<LNW_NT>(s2, red) * invC;
        wdg_ln_row<T, V>(gr, C, [&](int64_t c, int n, const WdgVec<T, V>& g) {
            const WdgVec<T, V> u = other(c, n);
            WdgVec<T, V> r;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float a = (float)g.e[j] * wdg_ln_param<T>(gamma, ptype, j < n ? c + j : c, 1.f);
                r.e[j] = (T)(rstd * (a - s1 - ((float)u.e[j] - mean) * rstd * s2));
            }
            wdg_ln_put<T, V>(dr + c, n, r);
        });
    }
}

// ---- parameter gradients -----------------------------------------------------------------------------------------------------------
// Partial sums [slice][dgamma | dbeta][C]: a block owns 256 V columns of one slice of the rows.
template <class T, int V>
__global__ void __launch_bounds__(256) wdg_layernorm_colsum_kernel(const T* __restrict__ dz, int64_t lddz, const T* __restrict__ x,
                                                                   int64_t ldx, const float* __restrict__ mean_rstd, float* part,
                                                                   int64_t P, int64_t C, int slices) {
    const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
    if (c >= C) return;
    const int n = (int)std::min<int64_t>(V, C - c);
    const int64_t per = (P + slices - 1) / slices, p0 = blockIdx.y * per, p1 = std::min<int64_t>(P, p0 + per);
    float sg[V], sb[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sg[j] = sb[j] = 0.f;
    for (int64_t p = p0; p < p1; ++p) {
        const float mean = mean_rstd[2 * p], rstd = mean_rstd[2 * p + 1];
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < n) {
                const float g = (float)dz[p * lddz + c + j];
                sg[j] += g * (((float)x[p * ldx + c + j] - mean) * rstd);
                sb[j] += g;
            }
    }
    float* row = part + (int64_t)blockIdx.y * 2 * C;
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j < n) {
            row[c + j] = sg[j];
            row[C + c + j] = sb[j];
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
    const int64_t col = (int64_t)blockIdx.x * CB + t % CB;
    float s = 0.f;
    if (col < 2 * C) {
#pragma unroll 8
        for (int r = t / CB; r < rows; r += SETS) s += part[(int64_t)r * 2 * C + col];
    }
    red[t] = s;
    __syncthreads();
    for (int o = SETS / 2; o > 0; o >>= 1) {
        if (t < o * CB) red[t] += red[t + o * CB];
        __syncthreads();
    }
    if (t < CB && col < 2 * C) {
        float* dst = col < C ? dgamma : dbeta;
        const int64_t c = col < C ? col : col - C;
        if (dst) dst[c] = (accumulate ? dst[c] : 0.f) + red[t];
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------------------------
struct LnBwdGeom {
    int slices;          // rows of the partial-sum table
};
static LnBwdGeom ln_bwd_geom(int64_t P, int64_t C, int type) {
    LnBwdGeom g;
    const int V = type == WDG_F32 ? 4 : 8;
    const int64_t tiles = (C + 256 * V - 1) / (256 * V);
    g.slices = (int)std::max<int64_t>(1, std::min<int64_t>((P + 15) / 16, std::max<int64_t>(1, 1024 / tiles)));
    return g;
}

static bool ln_types_ok(int type, int ptype) {
    return type >= WDG_F32 && type <= WDG_F16 && (ptype == WDG_F32 || ptype == type);
}
static const int64_t LN_MAX_C = 1ll << 24;      // (c / C and the sums' fp32 scale stay exact to rounding)

template <class T, int V>
static int ln_fwd_launch(const void* x, int64_t ldx, const void* gamma, const void* beta, int ptype, float eps, void* z, int64_t ldz,
                         float* mean_rstd, int64_t P, int64_t C, hipStream_t st) {
    const int blocks = (int)std::min<int64_t>(P, 4096);
    hipLaunchKernelGGL((wdg_layernorm_fwd_wide_kernel<T, V>), dim3(blocks), dim3(LNW_NT), 0, st, (const T*)x, ldx, gamma, beta, ptype, eps,
                       (T*)z, ldz, mean_rstd, P, C);
    WDG_LAUNCH_CHECK();
    return WDG_OK;
}

extern "C" int wdg_layernorm_fwd(const void* x, int64_t ldx, const void* gamma, const void* beta, float eps, void* z, int64_t ldz,
                                 float* mean_rstd, int64_t P, int64_t C, int type, int param_type, wdg_stream stream) {
    WDG_CHECK_ARG(ln_types_ok(type, param_type), "type: fp32, bf16 or fp16; parameters: fp32 or that type");
    WDG_CHECK_ARG(P >= 0 && C >= 1 && C <= LN_MAX_C, "bad sizes");
    if (P == 0) return WDG_OK;
    WDG_CHECK_ARG(x && z, "null argument");
    WDG_CHECK_ARG(ldx >= 0 && (P == 1 || ldz >= C), "output rows overlap");
    hipStream_t st = (hipStream_t)stream;
    if (type == WDG_F32) return ln_fwd_launch<float, 4>(x, ldx, gamma, beta, param_type, eps, z, ldz, mean_rstd, P, C, st);
    if (type == WDG_BF16) return ln_fwd_launch<__bf16, 8>(x, ldx, gamma, beta, param_type, eps, z, ldz, mean_rstd, P, C, st);
    return ln_fwd_launch<_Float16, 8>(x, ldx, gamma, beta, param_type, eps, z, ldz, mean_rstd, P, C, st);
}

extern "C" size_t wdg_layernorm_bwd_ws_bytes(int64_t P, int64_t C, int type) {
    if (P <= 0 || C <= 0 || C > LN_MAX_C || type < WDG_F32 || type > WDG_F16) return 0;
    return (size_t)ln_bwd_geom(P, C, type).slices * 2 * (size_t)C * sizeof(float);
}

static int ln_finish(const float* part, int rows, int64_t C, float* dgamma, float* dbeta, int accumulate, hipStream_t st) {
    if (2 * C <= 256)
        hipLaunchKernelGGL(wdg_layernorm_finish_kernel<16>, dim3((unsigned)((2 * C + 15) / 16)), dim3(1024), 0, st, part, rows, C, dgamma, dbeta, accumulate);
    else
        hipLaunchKernelGGL(wdg_layernorm_finish_kernel<64>, dim3((unsigned)((2 * C + 63) / 64)), dim3(1024), 0, st, part, rows, C, dgamma, dbeta, accumulate);
    WDG_LAUNCH_CHECK();
    return WDG_OK;
}

template <class T, int V>
static int ln_bwd_launch(const void* dz, int64_t lddz, const void* x, int64_t ldx, const float* mean_rstd, const void* gamma, int ptype,
                         void* dx, int64_t lddx, float* dgamma, float* dbeta, int accumulate, int64_t P, int64_t C, int type, float* part,
                         hipStream_t st) {
    if (dgamma || dbeta) {
        const int slices = P > 0 ? ln_bwd_geom(P, C, type).slices : 0;
        if (slices > 0) {
            hipLaunchKernelGGL((wdg_layernorm_colsum_kernel<T, V>), dim3((unsigned)((C + 256 * V - 1) / (256 * V)), slices), dim3(256), 0, st,
                               (const T*)dz, lddz, (const T*)x, ldx, mean_rstd, part, P, C, slices);
            WDG_LAUNCH_CHECK();
        }
        const int rc = ln_finish(part, slices, C, dgamma, dbeta, accumulate, st);
        if (rc != WDG_OK) return rc;
    }
    if (P == 0) return WDG_OK;
    hipLaunchKernelGGL((wdg_layernorm_bwd_wide_kernel<T, V>), dim3((unsigned)std::min<int64_t>(P, 4096)), dim3(LNW_NT), 0, st, (const T*)dz,
                       lddz, (const T*)x, ldx, mean_rstd, gamma, ptype, (T*)dx, lddx, P, C);
    WDG_LAUNCH_CHECK();
    return WDG_OK;
}

extern "C" int wdg_layernorm_bwd(const void* dz, int64_t lddz, const void* x, int64_t ldx, const float* mean_rstd, const void* gamma,
                                 void* dx, int64_t lddx, float* dgamma, float* dbeta, int accumulate, int64_t P, int64_t C, int type,
                                 int param_type, void* ws, size_t ws_bytes, wdg_stream stream) {
    WDG_CHECK_ARG(ln_types_ok(type, param_type), "type: fp32, bf16 or fp16; parameters: fp32 or that type");
    WDG_CHECK_ARG(P >= 0 && C >= 1 && C <= LN_MAX_C, "bad sizes");
    WDG_CHECK_ARG(P == 0 || (dz && x && mean_rstd && dx), "null argument");
    WDG_CHECK_ARG(lddz >= 0 && ldx >= 0 && (P <= 1 || lddx >= C), "gradient rows overlap");
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
