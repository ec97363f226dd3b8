// adamw.hip — AdamW over a list of tensors in one launch, states in 32 or 8 bits, with the global gradient norm that clips it.
// The formulas and the 8-bit format stand at wdg_adamw_step in wdgan.h.
//
// The list is cut into chunks of 4096 elements that never cross a tensor; a workgroup takes one chunk and finds everything about it in
// one record of the table (pointers already advanced), so that no search and no second dependent read stands before the data.
// A wave takes 256 consecutive elements at a time — four per lane —, which is one block of the 8-bit states: its two maxima are wave
// maxima and no other wave needs them.
//
// Bound: HBM.  64 M weights with bf16 gradients and copy: 278 us, 6.4 TB/s of exactly the bytes that the formulas name; 128 M with 8-bit
// states 345 us, 5.9 TB/s, at 93 vector instructions per element (decoding, exact root and quotient, two block maxima, two companding
// roots), which alone would take about 300.  The norm of 128 MB of gradients 27 us (4.7 TB/s).  A large copy reaches 5.3 TB/s.
#include "vec.h"
#include <algorithm>
#include <exception>
#include <math.h>
#include <utility>
#include <vector>

constexpr int AW_CHUNK = 4096;     // elements per record; AW_SMALL of them in short lists (aw_chunk_size)
constexpr int AW_SMALL = 1024;
constexpr int AW_BLOCK = 256;      // elements that share a scale of the 8-bit states
constexpr int AW_ALONE = 8;        // most chunks of a list whose step forms its norm in one launch
constexpr int AW_PARTS = 256;      // partial sums of the gradient norm: one for each thread of the step's workgroups

struct WdgAdamwChunk {
    void* p;
    const void* g;
    void* m;
    void* v;
    float* ms;
    float* vs;
    void* copy;
    int n;                                        // elements, 1 .. the batch's chunk size
    unsigned char p_type, g_type, copy_type, pad; // copy_type 0: no copy
    float decay;
    int pad2;
};
struct AwRange {
    uintptr_t begin, end;
    bool written;
};

struct wdg_adamw_batch {
    std::vector<WdgAdamwChunk> chunks;
    std::vector<AwRange> ranges;                  // the tensors' memory by address (gradients may share theirs) ...
    std::vector<uintptr_t> ends;                  // ... and the furthest end up to each of them
    int bits = 32;
    int chunk = AW_CHUNK;
    int64_t bytes = 0, grad_bytes = 0;            // of everything a step touches, of the gradients alone
    const WdgAdamwChunk* table = nullptr;         // device memory of the caller
};

// the step's numbers as the kernel takes them
struct WdgAdamwHyper {
    float b1, c1, b2, c2;                         // beta, 1 - beta
    float eps, lr_wd, lr;
    float lr_bc1, rbc2;                           // lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t), when t is known on the host
    double log_b1, log_b2;                        // ... otherwise they come from t in device memory
    const long long* step_dev;
    double grad_scale, max_norm;
    const double* parts;                          // partial sums of g^2, or NULL
    int nparts;
    int alone;                                    // > 0: so few chunks that every workgroup adds up the gradients of all of them itself
    float* norm;
};

// ---- four elements of a tensor, the missing ones of its last quad read as zero ----------------------------------------------------
template <bool STREAM = false, class T>
__device__ __forceinline__ f32x4 wdg_aw_load(const T* p, int n) {
    f32x4 r = {0.f, 0.f, 0.f, 0.f};
    if (n >= 4) {
        const WdgVec<T, 4> v = wdg_vec_load<T, 4, STREAM>(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = (float)v.e[j];
    } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (j < n) r[j] = (float)((const WDG_GLOBAL T*)p)[j];
    }
    return r;
}
template <bool STREAM = false, class T>
__device__ __forceinline__ void wdg_aw_store(T* p, int n, const f32x4& r) {
    if (n >= 4) {
        WdgVec<T, 4> v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v.e[j] = (T)r[j];
        wdg_vec_store<T, 4, STREAM>(p, v);
    } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (j < n) ((WDG_GLOBAL T*)p)[j] = (T)r[j];
    }
}

// largest of 64 lanes' unsigned values, in every lane: within rows of 16 lanes by DPP, the four rows through scalar registers
__device__ __forceinline__ unsigned wdg_wave_umax(unsigned v) {
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));     // quad_perm [1,0,3,2]
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));     // quad_perm [2,3,0,1]
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true));    // row_half_mirror
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true));    // row_mirror
    return max(max((unsigned)__builtin_amdgcn_readlane((int)v, 0), (unsigned)__builtin_amdgcn_readlane((int)v, 16)),
               max((unsigned)__builtin_amdgcn_readlane((int)v, 32), (unsigned)__builtin_amdgcn_readlane((int)v, 48)));
}
// the same for sums of doubles
template <int CTRL>
__device__ __forceinline__ double wdg_aw_dpp(double v) {
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    const i32x2 b = __builtin_bit_cast(i32x2, v);
    i32x2 r;
    r.x = __builtin_amdgcn_update_dpp(0, b.x, CTRL, 0xF, 0xF, true);
    r.y = __builtin_amdgcn_update_dpp(0, b.y, CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(double, r);
}
__device__ __forceinline__ double wdg_aw_lane(double v, int lane) {
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    const i32x2 b = __builtin_bit_cast(i32x2, v);
    i32x2 r;
    r.x = __builtin_amdgcn_readlane(b.x, lane);
    r.y = __builtin_amdgcn_readlane(b.y, lane);
    return __builtin_bit_cast(double, r);
}
__device__ __forceinline__ double wdg_aw_wave_sum(double v) {
    v += wdg_aw_dpp<0xB1>(v);
    v += wdg_aw_dpp<0x4E>(v);
    v += wdg_aw_dpp<0x141>(v);
    v += wdg_aw_dpp<0x140>(v);
    return (wdg_aw_lane(v, 0) + wdg_aw_lane(v, 16)) + (wdg_aw_lane(v, 32) + wdg_aw_lane(v, 48));
}
// A block's scale from the largest bit pattern of its magnitudes (as integers: above infinity come the NaNs, which a float maximum would
// drop).  inv = 1 / scale, 0 where the block holds zeros alone; a block that is not finite gets a NaN for its scale.
// First moments below 2^-126 count as zero: the scale's reciprocal would not be a number.  The scale of second moments is 2^-94 at least,
// so that code 1, a 255^4th of it, is a normal number: what is above zero does not read as zero.
template <bool SECOND>
__device__ __forceinline__ float wdg_aw_scale(unsigned bits, float& inv) {
    constexpr unsigned least = SECOND ? (127u - 94u) << 23 : 1u << 23;
    if (bits >= 0x7f800000u) {
        inv = 0.f;
        return __builtin_nanf("");
    }
    if (SECOND && bits != 0) bits = max(bits, least);
    if (bits < least) {
        inv = 0.f;
        return 0.f;
    }
    const float s = __builtin_bit_cast(float, bits);
    inv = 1.f / s;
    return s;
}

// a chunk's share of the sum of g^2, per thread of 256; fp64, since a square leaves fp32's range where the gradient itself does not
template <int CHUNK, bool STREAM, class GT>
__device__ __forceinline__ double wdg_aw_sumsq(const GT* g, int n) {
    const int t = (int)(threadIdx.x & 255) * 4;
    f32x4 v[CHUNK / 1024];
    if (n == CHUNK) {
#pragma unroll
        for (int i = 0; i < CHUNK / 1024; ++i) v[i] = wdg_aw_load<STREAM>(g + i * 1024 + t, 4);
    } else {
#pragma unroll
        for (int i = 0; i < CHUNK / 1024; ++i) v[i] = wdg_aw_load<STREAM>(g + i * 1024 + t, n - i * 1024 - t);
    }
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < CHUNK / 1024; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s += (double)v[i][j] * (double)v[i][j];
    return s;
}
// clipping: the gradients' factor grad_scale c, the same bits in every workgroup (all add the same numbers in the same order); false
// where the norm is not finite in fp32.  All threads of the workgroup call it once.  `part`: this thread's partial sum, asked for at the start.
__device__ __forceinline__ bool wdg_aw_clip(const WdgAdamwHyper& h, double part, double* red, float& gs) {
    gs = (float)h.grad_scale;
    if (!h.parts && !h.alone) return true;
    const double s = wdg_aw_wave_sum(part);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    const double norm = h.grad_scale * sqrt((red[0] + red[1]) + (red[2] + red[3]));
    if (h.norm && blockIdx.x == 0 && threadIdx.x == 0) h.norm[0] = (float)norm;
    if (!((float)norm < INFINITY)) return false;             // (as it is handed out: the caller sees which steps changed nothing)
    gs = (float)(h.grad_scale * (h.max_norm / fmax(norm, h.max_norm)));
    return true;
}

// One chunk.  FULL: all its elements are there, so every request is issued without a condition and before the first answer is used;
// else the tensor ends inside, and a thread takes one quad after the other and looks at what is left.  The first requests go out before the
// workgroup adds up the norm.
template <int BITS, int CHUNK, bool STREAM, class PT, class GT, bool FULL>
__device__ __forceinline__ void wdg_aw_chunk(const WdgAdamwChunk& q, const WdgAdamwHyper& h, double part, double* red, float lr_bc1, float rbc2) {
    constexpr int QUADS = CHUNK / 1024, UN = FULL ? QUADS : 1;
    // the decay's factor 1 - lr weight_decay d as two numbers: alone the first is a multiple of 2^-24, and every step of a run would decay by
    // the same wrong amount (lr weight_decay = 4e-8 by half too much, 2e-8 not at all)
    const float lwd = h.lr_wd * q.decay, keep = 1.f - lwd, keep_rest = (1.f - keep) - lwd;
    PT* p = static_cast<PT*>(q.p);
    const GT* g = static_cast<const GT*>(q.g);
    const int lane = threadIdx.x & 63;
    f32x4 w[UN], gr[UN], m[UN], v[UN];
    unsigned cm[UN], cv[UN];
    float sm[UN], sv[UN], gs;
    auto behind = [&](int i) { return !FULL && i * 1024 + ((int)threadIdx.x & ~63) * 4 >= q.n; };      // (the wave's whole block lies behind the tensor)
    auto fetch = [&](int i) {
        if (behind(i)) return;
#pragma unroll
        for (int k = 0; k < UN; ++k) {
            const int e = ((i + k) * 256 + (int)threadIdx.x) * 4, n = FULL ? 4 : q.n - e;      // (n: elements from here on, maybe none)
            w[k] = wdg_aw_load<STREAM>(p + e, n);
            gr[k] = wdg_aw_load<STREAM>(g + e, n);
            if constexpr (BITS == 32) {
                m[k] = wdg_aw_load<STREAM>(static_cast<const float*>(q.m) + e, n);
                v[k] = wdg_aw_load<STREAM>(static_cast<const float*>(q.v) + e, n);
            } else {
                cm[k] = wdg_vec_load<unsigned, 1, STREAM>(static_cast<const unsigned*>(q.m) + (e >> 2)).e[0];
                cv[k] = wdg_vec_load<unsigned, 1, STREAM>(static_cast<const unsigned*>(q.v) + (e >> 2)).e[0];
                sm[k] = ((const WDG_GLOBAL float*)q.ms)[e / AW_BLOCK];
                sv[k] = ((const WDG_GLOBAL float*)q.vs)[e / AW_BLOCK];
            }
        }
    };
    fetch(0);
    if (!wdg_aw_clip(h, part, red, gs)) return;
#pragma unroll 1
    for (int i = 0;; fetch(i)) {
        if (behind(i)) return;
#pragma unroll
        for (int k = 0; k < UN; ++k) {
            const int e = ((i + k) * 256 + (int)threadIdx.x) * 4, n = FULL ? 4 : q.n - e;
            if constexpr (BITS == 8) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float a = (float)(signed char)(cm[k] >> (8 * j)), b = (float)((cv[k] >> (8 * j)) & 255u) * (1.f / 255.f);
                    m[k][j] = a * fabsf(a) * (sm[k] * (1.f / (127.f * 127.f)));
                    v[k][j] = (b * b) * (b * b) * sv[k];
                }
            }
            unsigned tm = 0, tv = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float gj = gr[k][j] * gs;
                const float a = h.b1 * m[k][j] + h.c1 * gj, b = h.b2 * v[k][j] + h.c2 * (gj * gj);
                m[k][j] = a;
                v[k][j] = b;
                // (the small product of a finite weight: an infinite one stays infinite)
                const float rest = fmaf(__builtin_amdgcn_fmed3f(w[k][j], -3.4028235e38f, 3.4028235e38f), keep_rest, -lr_bc1 * (a / (sqrtf(b) * rbc2 + h.eps)));
                w[k][j] = fmaf(w[k][j], keep, rest);
                if constexpr (BITS == 8) {               // (from the scalars: a bit cast of a vector's element would take element 0)
                    tm = max(tm, j < n ? __builtin_bit_cast(unsigned, a) & 0x7fffffffu : 0u);
                    tv = max(tv, j < n ? __builtin_bit_cast(unsigned, b) & 0x7fffffffu : 0u);
                }
            }
            wdg_aw_store<STREAM>(p + e, n, w[k]);
            if (q.copy_type == WDG_BF16) wdg_aw_store<STREAM>(static_cast<__bf16*>(q.copy) + e, n, w[k]);
            else if (q.copy_type == WDG_F16) wdg_aw_store<STREAM>(static_cast<_Float16*>(q.copy) + e, n, w[k]);
            if constexpr (BITS == 32) {
                wdg_aw_store<STREAM>(static_cast<float*>(q.m) + e, n, m[k]);
                wdg_aw_store<STREAM>(static_cast<float*>(q.v) + e, n, v[k]);
            } else {
                float im, iv;
                const float nm = wdg_aw_scale<false>(wdg_wave_umax(tm), im), nv = wdg_aw_scale<true>(wdg_wave_umax(tv), iv);
                unsigned om = 0, ov = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (j >= n) continue;
                    // both companding roots on the hardware square root (one unit in the last place of a value that is rounded to
                    // 1 / 127 or 1 / 255): only a value that close to the border between two codes can take the other one
                    const float a = rintf(127.f * __builtin_amdgcn_sqrtf(fabsf(m[k][j]) * im));
                    // (v itself decides whether there is one: its quotient to the block's largest may be below fp32's range)
                    const float b = v[k][j] > 0.f ? fmaxf(rintf(255.f * __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(v[k][j] * iv))), 1.f) : 0.f;
                    const int ai = im > 0.f ? (int)(m[k][j] < 0.f ? -a : a) : 0, bi = iv > 0.f ? (int)b : 0;
                    om |= ((unsigned)ai & 255u) << (8 * j);
                    ov |= ((unsigned)bi & 255u) << (8 * j);
                }
                wdg_vec_store<unsigned, 1, STREAM>(static_cast<unsigned*>(q.m) + (e >> 2), {{om}});
                wdg_vec_store<unsigned, 1, STREAM>(static_cast<unsigned*>(q.v) + (e >> 2), {{ov}});
                if (lane == 0) {
                    ((WDG_GLOBAL float*)q.ms)[e / AW_BLOCK] = nm;
                    ((WDG_GLOBAL float*)q.vs)[e / AW_BLOCK] = nv;
                }
            }
        }
        i += UN;
        if (i >= QUADS) return;
    }
}

template <int BITS, int CHUNK, bool STREAM, class PT, class GT>
__device__ __forceinline__ void wdg_aw_by_size(const WdgAdamwChunk& q, const WdgAdamwHyper& h, double part, double* red, float lr_bc1, float rbc2) {
    if (q.n == CHUNK) wdg_aw_chunk<BITS, CHUNK, STREAM, PT, GT, true>(q, h, part, red, lr_bc1, rbc2);
    else wdg_aw_chunk<BITS, CHUNK, STREAM, PT, GT, false>(q, h, part, red, lr_bc1, rbc2);
}
template <int BITS, int CHUNK, bool STREAM, class PT>
__device__ __forceinline__ void wdg_aw_by_grad(const WdgAdamwChunk& q, const WdgAdamwHyper& h, double part, double* red, float lr_bc1, float rbc2) {
    if (q.g_type == WDG_F32) wdg_aw_by_size<BITS, CHUNK, STREAM, PT, float>(q, h, part, red, lr_bc1, rbc2);
    else if (q.g_type == WDG_BF16) wdg_aw_by_size<BITS, CHUNK, STREAM, PT, __bf16>(q, h, part, red, lr_bc1, rbc2);
    else wdg_aw_by_size<BITS, CHUNK, STREAM, PT, _Float16>(q, h, part, red, lr_bc1, rbc2);
}

template <int BITS, int CHUNK, bool STREAM>
__global__ void __launch_bounds__(256) wdg_adamw_kernel(const WdgAdamwChunk* __restrict__ table, const WdgAdamwHyper h) {
    __shared__ double red[4];
    double part = h.parts && (int)threadIdx.x < h.nparts ? h.parts[threadIdx.x] : 0.0;
    const WdgAdamwChunk q = table[blockIdx.x];
    if constexpr (CHUNK == AW_SMALL) {
        for (int c = 0; c < h.alone; ++c) {
            const WdgAdamwChunk& o = table[c];
            if (o.g_type == WDG_F32) part += wdg_aw_sumsq<CHUNK, false>(static_cast<const float*>(o.g), o.n);
            else if (o.g_type == WDG_BF16) part += wdg_aw_sumsq<CHUNK, false>(static_cast<const __bf16*>(o.g), o.n);
            else part += wdg_aw_sumsq<CHUNK, false>(static_cast<const _Float16*>(o.g), o.n);
        }
    }
    float lr_bc1 = h.lr_bc1, rbc2 = h.rbc2;
    if (h.step_dev) {
        // 1 - beta^t = -expm1(t log beta): the difference keeps its digits when beta^t is close to 1
        const double t = (double)*h.step_dev;
        lr_bc1 = h.lr / -expm1f((float)(t * h.log_b1));
        rbc2 = 1.f / sqrtf(-expm1f((float)(t * h.log_b2)));
    }
    if (q.p_type == WDG_F32) wdg_aw_by_grad<BITS, CHUNK, STREAM, float>(q, h, part, red, lr_bc1, rbc2);
    else if (q.p_type == WDG_BF16) wdg_aw_by_grad<BITS, CHUNK, STREAM, __bf16>(q, h, part, red, lr_bc1, rbc2);
    else wdg_aw_by_grad<BITS, CHUNK, STREAM, _Float16>(q, h, part, red, lr_bc1, rbc2);
}

// ---- sum of g^2 over all chunks ------------------------------------------------------------------------------------------------------
// Four chunks at a time per workgroup (256 threads each), as many workgroups as the chip holds: the launch reads one tensor, and what it
// needs is requests in flight.
template <int CHUNK, bool STREAM>
__global__ void __launch_bounds__(1024) wdg_adamw_sumsq_kernel(const WdgAdamwChunk* __restrict__ table, int chunks, double* parts) {
    constexpr int R = AW_CHUNK / CHUNK;                   // records at a time
    __shared__ double red[16];
    double s = 0.0;
    for (int c0 = (blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 8)) * R; c0 < chunks; c0 += gridDim.x * (4 * R)) {
        const void* g[R];
        int n[R], type[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const WdgAdamwChunk& q = table[min(c0 + r, chunks - 1)];
            g[r] = q.g;
            n[r] = c0 + r < chunks ? q.n : 0;
            type[r] = q.g_type;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (type[r] == WDG_F32) s += wdg_aw_sumsq<CHUNK, STREAM>(static_cast<const float*>(g[r]), n[r]);
            else if (type[r] == WDG_BF16) s += wdg_aw_sumsq<CHUNK, STREAM>(static_cast<const __bf16*>(g[r]), n[r]);
            else s += wdg_aw_sumsq<CHUNK, STREAM>(static_cast<const _Float16*>(g[r]), n[r]);
        }
    }
    s = wdg_aw_wave_sum(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double total = 0.0;
#pragma unroll
        for (int w = 0; w < 16; ++w) total += red[w];
        parts[blockIdx.x] = total;
    }
}
__global__ void __launch_bounds__(256) wdg_adamw_norm_kernel(const double* __restrict__ parts, int nparts, double scale, float* norm) {
    __shared__ double red[4];
    double s = 0.0;
    for (int i = threadIdx.x; i < nparts; i += 256) s += parts[i];
    s = wdg_aw_wave_sum(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) norm[0] = (float)(scale * sqrt((red[0] + red[1]) + (red[2] + red[3])));
}

// ---- the values behind 8-bit states: 16 codes per thread, blockIdx.y 0 the first moment, 1 the second ----------------------------
template <class T>
__global__ void __launch_bounds__(256) wdg_adamw_moments_kernel(const unsigned char* m, const float* ms, const unsigned char* v, const float* vs,
                                                                T* mo, T* vo, long long sixteens) {
    const bool second = blockIdx.y == 1;
    T* out = second ? vo : mo;
    if (!out) return;
    const unsigned char* codes = second ? v : m;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < sixteens; i += (long long)gridDim.x * 256) {
        const WdgVec<unsigned, 4> c = wdg_vec_load<unsigned, 4>(reinterpret_cast<const unsigned*>(codes) + 4 * i);
        const float s = (second ? vs : ms)[i / (AW_BLOCK / 16)];
        const float s1 = s * (1.f / (127.f * 127.f));
        WdgVec<T, 16> r;
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float a = (float)(signed char)(c.e[k] >> (8 * j)), b = (float)((c.e[k] >> (8 * j)) & 255u) * (1.f / 255.f);
                r.e[4 * k + j] = (T)(second ? (b * b) * (b * b) * s : a * fabsf(a) * s1);
            }
        wdg_vec_store<T, 16>(out + 16 * i, r);
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------------------------
static int aw_bytes(int type) { return type == WDG_F32 ? 4 : 2; }
static bool aw_aligned(const void* p, int a) { return ((uintptr_t)p & (uintptr_t)(a - 1)) == 0; }

// NULL, or what is wrong with tensor t
static const char* aw_check(const wdg_adamw_tensor& t, int bits) {
    if (t.n < 0) return "negative size";
    if (t.p_type < WDG_F32 || t.p_type > WDG_F16 || t.g_type < WDG_F32 || t.g_type > WDG_F16) return "unknown type";
    if (t.copy && t.copy_type != WDG_BF16 && t.copy_type != WDG_F16) return "the copy is bf16 or fp16";
    if (!(t.decay >= 0.f) || t.decay > 3.4e38f) return "decay factor";
    if (t.n == 0) return nullptr;
    if (!t.p || !t.g || !t.m || !t.v || (bits == 8 && (!t.m_scale || !t.v_scale))) return "null pointer";
    if (!aw_aligned(t.p, aw_bytes(t.p_type)) || !aw_aligned(t.g, aw_bytes(t.g_type)) || !aw_aligned(t.copy, 2) || !aw_aligned(t.m, 4) ||
        !aw_aligned(t.v, 4) || !aw_aligned(t.m_scale, 4) || !aw_aligned(t.v_scale, 4))
        return "not aligned to its element";
    return nullptr;
}

// Lists of fewer than 4096 chunks of 4096 (16 M elements) in chunks of 1024: more workgroups than the chip holds at once, and one request
// per tensor and thread, hide a chunk's latency better (us of an unclipped fp32 step with 1024 / 4096, 32-bit states: 0.2 M elements
// 3.5 / 4.6, 2 M 10.5 / 13.8, 8 M 43.7 / 45.7; 8-bit: 3.8 / 6.4, 9.5 / 13.0, 23 / 27).  Above, the table and the norm that every workgroup
// of a clipped step adds up cost what that gains (16 M, 8-bit, clipped: 68 / 66).
static int aw_chunk_size(int64_t chunks) { return chunks < 4096 ? AW_SMALL : AW_CHUNK; }

// A step whose tensors leave no room in the chip's last-level cache (256 MiB) is streamed past it: nothing of it would be there at the
// next step.  us without / with, 32-bit states: 8 M fp32 (122 MiB) 43 / 38, 16 M 86 / 74, 128 M 681 / 627; 8-bit: 16 M (152 MiB) 50 / 45,
// 128 M 383 / 351; smaller ones stay: 4 M (61 MiB) 18.5 / 20.4.
static bool aw_stream_step(const wdg_adamw_batch* b) { return b->bytes >= 96ll << 20; }
// The norm's pass leaves the gradients in the cache for the step where they fit: 32 M fp32 (122 MiB), clipped, 178 us with streaming and
// 159 without; 128 M (488 MiB) 703 and 792.
static bool aw_stream_norm(const wdg_adamw_batch* b) { return b->grad_bytes >= 192ll << 20; }

static int aw_create(wdg_adamw_batch** out, const wdg_adamw_tensor* tensors, int n, int bits) {
    std::vector<AwRange> ranges;
    int64_t chunks = 0, total = 0, grads = 0;
    for (int i = 0; i < n; ++i) {
        const wdg_adamw_tensor& t = tensors[i];
        if (const char* why = aw_check(t, bits)) {
            wdg_set_error("wdg_adamw_create: tensor %d: %s", i, why);
            return WDG_ERR_ARG;
        }
        if (t.n == 0) continue;
        const int64_t blocks = (t.n + AW_BLOCK - 1) / AW_BLOCK;
        auto add = [&](const void* p, int64_t bytes, bool written) {
            if (p) ranges.push_back({(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes, written});
            if (p) total += bytes;
        };
        add(t.p, t.n * aw_bytes(t.p_type), true);
        add(t.g, t.n * aw_bytes(t.g_type), false);
        grads += t.n * aw_bytes(t.g_type);
        add(t.copy, t.n * 2, true);
        add(t.m, bits == 8 ? blocks * AW_BLOCK : t.n * 4, true);
        add(t.v, bits == 8 ? blocks * AW_BLOCK : t.n * 4, true);
        if (bits == 8) {
            add(t.m_scale, blocks * 4, true);
            add(t.v_scale, blocks * 4, true);
        }
        chunks += (t.n + AW_CHUNK - 1) / AW_CHUNK;
    }
    if (chunks > 0x7fffffff) {
        wdg_set_error("wdg_adamw_create: more than 2^31 chunks of %d elements", AW_CHUNK);
        return WDG_ERR_ARG;
    }
    // in address order, a range may only begin where every written one before it — and, if it is written itself, every one — has ended
    std::sort(ranges.begin(), ranges.end(), [](const AwRange& a, const AwRange& b) { return a.begin < b.begin; });
    uintptr_t end_written = 0, end_any = 0;
    for (const AwRange& r : ranges) {
        if (r.begin < (r.written ? end_any : end_written)) {
            wdg_set_error("wdg_adamw_create: tensors overlap (the same one twice, a gradient over a weight or a state of two tensors)");
            return WDG_ERR_ARG;
        }
        end_any = std::max(end_any, r.end);
        if (r.written) end_written = std::max(end_written, r.end);
    }
    wdg_adamw_batch* b = new wdg_adamw_batch();
    b->bits = bits;
    b->chunk = aw_chunk_size(chunks);
    b->bytes = total;
    b->grad_bytes = grads;
    try {
        b->chunks.reserve((size_t)(chunks * (AW_CHUNK / b->chunk)));
        b->ends.reserve(ranges.size());
    } catch (...) {
        delete b;
        throw;
    }
    for (int i = 0; i < n; ++i) {
        const wdg_adamw_tensor& t = tensors[i];
        for (int64_t e = 0; e < t.n; e += b->chunk) {
            WdgAdamwChunk q;
            memset(&q, 0, sizeof(q));
            q.p = (char*)t.p + e * aw_bytes(t.p_type);
            q.g = (const char*)t.g + e * aw_bytes(t.g_type);
            q.m = (char*)t.m + e * (bits == 8 ? 1 : 4);
            q.v = (char*)t.v + e * (bits == 8 ? 1 : 4);
            q.ms = bits == 8 ? t.m_scale + e / AW_BLOCK : nullptr;
            q.vs = bits == 8 ? t.v_scale + e / AW_BLOCK : nullptr;
            q.copy = t.copy ? (char*)t.copy + e * 2 : nullptr;
            q.n = (int)std::min<int64_t>(b->chunk, t.n - e);
            q.p_type = (unsigned char)t.p_type;
            q.g_type = (unsigned char)t.g_type;
            q.copy_type = t.copy ? (unsigned char)t.copy_type : 0;
            q.decay = t.decay;
            b->chunks.push_back(q);
        }
    }
    for (const AwRange& r : ranges) b->ends.push_back(std::max(b->ends.empty() ? 0 : b->ends.back(), r.end));
    b->ranges = std::move(ranges);
    *out = b;
    return WDG_OK;
}

// whether `bytes` at p meet a tensor of the list
static bool aw_meets(const wdg_adamw_batch* b, const void* p, size_t bytes) {
    if (!p) return false;
    const uintptr_t begin = (uintptr_t)p, end = begin + bytes;
    const auto behind = std::lower_bound(b->ranges.begin(), b->ranges.end(), end, [](const AwRange& r, uintptr_t e) { return r.begin < e; });
    return behind != b->ranges.begin() && b->ends[behind - b->ranges.begin() - 1] > begin;
}
static bool aw_apart(const void* p, size_t np, const void* q, size_t nq) {
    return !p || !q || (uintptr_t)p + np <= (uintptr_t)q || (uintptr_t)q + nq <= (uintptr_t)p;
}
// what a call writes and reads beside the list's tensors has to be memory of its own: NULL, or what is not
static const char* aw_beside(const wdg_adamw_batch* b, const void* norm, const void* step_dev, const void* scratch) {
    if (aw_meets(b, norm, sizeof(float))) return "the norm overlaps a tensor of the list";
    if (aw_meets(b, step_dev, sizeof(int64_t))) return "the step count overlaps a tensor of the list";
    if (aw_meets(b, scratch, AW_PARTS * sizeof(double))) return "the scratch overlaps a tensor of the list";
    if (!aw_apart(norm, sizeof(float), scratch, AW_PARTS * sizeof(double)) || !aw_apart(norm, sizeof(float), step_dev, sizeof(int64_t)) ||
        !aw_apart(step_dev, sizeof(int64_t), scratch, AW_PARTS * sizeof(double)))
        return "norm, step count and scratch overlap";
    return nullptr;
}

extern "C" int wdg_adamw_create(wdg_adamw_batch** out, const wdg_adamw_tensor* tensors, int n, int state_bits) {
    WDG_CHECK_ARG(out && n >= 0 && (tensors || n == 0), "bad argument");
    WDG_CHECK_ARG(state_bits == 32 || state_bits == 8, "states are held in 32 or 8 bits");
    try {
        return aw_create(out, tensors, n, state_bits);
    } catch (const std::exception& e) {
        wdg_set_error("wdg_adamw_create: %s", e.what());
        return WDG_ERR_ARG;
    }
}

extern "C" size_t wdg_adamw_table_bytes(const wdg_adamw_batch* b) { return b ? b->chunks.size() * sizeof(WdgAdamwChunk) : 0; }

extern "C" int wdg_adamw_bind(wdg_adamw_batch* b, void* table, size_t table_bytes, wdg_stream stream) {
    WDG_CHECK_ARG(b, "null batch");
    if (b->chunks.empty()) return WDG_OK;
    WDG_CHECK_ARG(table && aw_aligned(table, 16) && table_bytes >= wdg_adamw_table_bytes(b), "table: wdg_adamw_table_bytes() of device memory, 16-byte aligned");
    WDG_HIP(hipMemcpyAsync(table, b->chunks.data(), wdg_adamw_table_bytes(b), hipMemcpyHostToDevice, (hipStream_t)stream));
    WDG_HIP(hipStreamSynchronize((hipStream_t)stream));
    b->table = (const WdgAdamwChunk*)table;
    return WDG_OK;
}

extern "C" int wdg_adamw_destroy(wdg_adamw_batch* b) {
    delete b;
    return WDG_OK;
}

extern "C" size_t wdg_adamw_scratch_bytes(void) { return AW_PARTS * sizeof(double); }

static int aw_parts(const wdg_adamw_batch* b) {
    const size_t each = 4 * (AW_CHUNK / b->chunk);        // chunks that a workgroup takes at a time
    return (int)std::min<size_t>(AW_PARTS, (b->chunks.size() + each - 1) / each);
}

static int aw_sumsq(const wdg_adamw_batch* b, double* parts, hipStream_t st) {
    if (aw_parts(b) == 0) return WDG_OK;
    const auto kernel = b->chunk == AW_SMALL ? wdg_adamw_sumsq_kernel<AW_SMALL, false>
                        : aw_stream_norm(b) ? wdg_adamw_sumsq_kernel<AW_CHUNK, true> : wdg_adamw_sumsq_kernel<AW_CHUNK, false>;
    hipLaunchKernelGGL(kernel, dim3(aw_parts(b)), dim3(1024), 0, st, b->table, (int)b->chunks.size(), parts);
    WDG_LAUNCH_CHECK();
    return WDG_OK;
}

static int aw_norm(const wdg_adamw_batch* b, double scale, float* norm, const double* parts, hipStream_t st) {
    hipLaunchKernelGGL(wdg_adamw_norm_kernel, dim3(1), dim3(256), 0, st, parts, aw_parts(b), scale, norm);
    WDG_LAUNCH_CHECK();
    return WDG_OK;
}

extern "C" int wdg_adamw_grad_norm(const wdg_adamw_batch* b, double grad_scale, float* norm, void* scratch, size_t scratch_bytes,
                                   wdg_stream stream) {
    WDG_CHECK_ARG(b && norm, "null argument");
    WDG_CHECK_ARG(grad_scale >= 0.0 && grad_scale < INFINITY, "gradient scale");
    if (!scratch || !aw_aligned(scratch, 8) || scratch_bytes < wdg_adamw_scratch_bytes()) {
        wdg_set_error("wdg_adamw_grad_norm: scratch too small or not aligned");
        return WDG_ERR_WORKSPACE;
    }
    const char* beside = aw_beside(b, norm, nullptr, scratch);
    WDG_CHECK_ARG(!beside, beside);
    WDG_CHECK_ARG(b->chunks.empty() || b->table, "wdg_adamw_bind has not been called");
    const int rc = aw_sumsq(b, (double*)scratch, (hipStream_t)stream);
    return rc != WDG_OK ? rc : aw_norm(b, grad_scale, norm, (const double*)scratch, (hipStream_t)stream);
}

template <int BITS>
static auto aw_step_kernel(const wdg_adamw_batch* b) {
    if (b->chunk == AW_SMALL) return aw_stream_step(b) ? wdg_adamw_kernel<BITS, AW_SMALL, true> : wdg_adamw_kernel<BITS, AW_SMALL, false>;
    return aw_stream_step(b) ? wdg_adamw_kernel<BITS, AW_CHUNK, true> : wdg_adamw_kernel<BITS, AW_CHUNK, false>;
}

extern "C" int wdg_adamw_step(const wdg_adamw_batch* b, const wdg_adamw_args* a, void* scratch, size_t scratch_bytes, wdg_stream stream) {
    WDG_CHECK_ARG(b && a, "null argument");
    WDG_CHECK_ARG(a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0, "beta1 and beta2 have to be in [0, 1)");
    WDG_CHECK_ARG(a->eps >= 0.0 && a->lr >= 0.0 && a->weight_decay >= 0.0 && a->grad_scale >= 0.0 && a->eps < INFINITY && a->lr < INFINITY &&
                      a->weight_decay < INFINITY && a->grad_scale < INFINITY && a->max_norm < INFINITY, "lr, eps, weight decay and gradient scale: finite, not negative");
    WDG_CHECK_ARG(a->step_dev || a->step >= 1, "steps count from 1");
    const bool clip = a->max_norm > 0.0;
    hipStream_t st = (hipStream_t)stream;
    if (clip && (!scratch || !aw_aligned(scratch, 8) || scratch_bytes < wdg_adamw_scratch_bytes())) {
        wdg_set_error("wdg_adamw_step: scratch too small or not aligned");
        return WDG_ERR_WORKSPACE;
    }
    const char* beside = aw_beside(b, clip ? a->norm : nullptr, a->step_dev, clip ? scratch : nullptr);
    WDG_CHECK_ARG(!beside, beside);
    WDG_CHECK_ARG(b->chunks.empty() || b->table, "wdg_adamw_bind has not been called");
    if (b->chunks.empty()) return clip && a->norm ? aw_norm(b, 0.0, a->norm, (const double*)scratch, st) : WDG_OK;
    // up to 8 chunks of 1024: one launch instead of two (3000 elements: 4.0 us instead of 5.5 in a graph, 6.8 instead of 9.6 a call; each
    // chunk more adds 0.3 us to what every workgroup does by itself)
    const bool alone = b->chunk == AW_SMALL && b->chunks.size() <= AW_ALONE;
    if (clip && !alone) {
        const int rc = aw_sumsq(b, (double*)scratch, st);
        if (rc != WDG_OK) return rc;
    }
    WdgAdamwHyper h;
    memset(&h, 0, sizeof(h));
    h.b1 = (float)a->beta1;
    h.c1 = (float)(1.0 - a->beta1);
    h.b2 = (float)a->beta2;
    h.c2 = (float)(1.0 - a->beta2);
    h.eps = (float)a->eps;
    h.lr = (float)a->lr;
    h.lr_wd = (float)(a->lr * a->weight_decay);
    h.step_dev = (const long long*)a->step_dev;
    if (a->step_dev) {
        h.log_b1 = log(a->beta1);                  // (beta = 0: -inf, and 1 - beta^t = 1)
        h.log_b2 = log(a->beta2);
    } else {
        h.lr_bc1 = (float)(a->lr / (1.0 - pow(a->beta1, (double)a->step)));
        h.rbc2 = (float)(1.0 / sqrt(1.0 - pow(a->beta2, (double)a->step)));
    }
    h.grad_scale = a->grad_scale;
    if (clip) {
        h.max_norm = a->max_norm;
        h.parts = alone ? nullptr : (const double*)scratch;
        h.nparts = alone ? 0 : aw_parts(b);
        h.alone = alone ? (int)b->chunks.size() : 0;
        h.norm = a->norm;
    }
    const dim3 grid((unsigned)b->chunks.size());
    const auto kernel = b->bits == 32 ? aw_step_kernel<32>(b) : aw_step_kernel<8>(b);
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, b->table, h);
    WDG_LAUNCH_CHECK();
    return WDG_OK;
}

extern "C" int wdg_adamw_moments(const void* m, const float* m_scale, const void* v, const float* v_scale, int64_t blocks, void* m_out,
                                 void* v_out, int out_type, wdg_stream stream) {
    WDG_CHECK_ARG(blocks >= 0 && out_type >= WDG_F32 && out_type <= WDG_F16, "bad argument");
    if (blocks == 0 || (!m_out && !v_out)) return WDG_OK;
    WDG_CHECK_ARG((!m_out || (m && m_scale)) && (!v_out || (v && v_scale)), "null argument");
    WDG_CHECK_ARG(aw_aligned(m, 4) && aw_aligned(v, 4) && aw_aligned(m_out, aw_bytes(out_type)) && aw_aligned(v_out, aw_bytes(out_type)), "alignment");
    const size_t n = (size_t)blocks * AW_BLOCK, out = n * aw_bytes(out_type), scales = (size_t)blocks * sizeof(float);
    bool apart = aw_apart(m_out, out, v_out, out);
    for (const void* o : {m_out, v_out})
        apart = apart && aw_apart(o, out, m, n) && aw_apart(o, out, v, n) && aw_apart(o, out, m_scale, scales) && aw_apart(o, out, v_scale, scales);
    WDG_CHECK_ARG(apart, "the moments read out overlap each other or the states");
    const long long sixteens = blocks * (AW_BLOCK / 16);
    const dim3 grid((unsigned)std::min<long long>((sixteens + 255) / 256, 16384), 2);
    hipStream_t st = (hipStream_t)stream;
    const unsigned char *mc = (const unsigned char*)m, *vc = (const unsigned char*)v;
    if (out_type == WDG_F32) hipLaunchKernelGGL(wdg_adamw_moments_kernel<float>, grid, dim3(256), 0, st, mc, m_scale, vc, v_scale, (float*)m_out, (float*)v_out, sixteens);
    else if (out_type == WDG_BF16) hipLaunchKernelGGL(wdg_adamw_moments_kernel<__bf16>, grid, dim3(256), 0, st, mc, m_scale, vc, v_scale, (__bf16*)m_out, (__bf16*)v_out, sixteens);
    else hipLaunchKernelGGL(wdg_adamw_moments_kernel<_Float16>, grid, dim3(256), 0, st, mc, m_scale, vc, v_scale, (_Float16*)m_out, (_Float16*)v_out, sixteens);
    WDG_LAUNCH_CHECK();
    return WDG_OK;
}
