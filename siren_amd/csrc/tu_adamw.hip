// tu_adamw.hip — one AdamW step over a list of tensors, with the moments in 32 bits or in 8.
//
//   g' = c g, c = min(1, max_norm / (||g|| + 1e-6)) over all tensors (c = 1 without a max_norm)
//   m  = m + (1 - b1) (g' - m),  v = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// The moments are flat, each tensor padded to a multiple of 128 elements. With 8 bits they are e4m3 codes of m and of
// u = sqrt(v) (the root halves v's range in powers of two: 2^-9 .. 448 then covers 5e10 : 1 within a block), with one
// scale 2^(byte - 127) per 128. Rounding to the nearest would leave a moment where it is as long as a step moves it by
// less than half a code (b2 = 0.999 moves u by 0.05 %, half a code is 3 to 6 %), so the codes are rounded up or down
// at random with the right mean, by 16 bits of splitmix64(seed, t, element): the step's outcome is a function of its
// inputs. The update of p uses the moments before they are rounded.
//
// Bytes bound it: 28 a parameter with fp32 moments, 16 with 8-bit ones (p read and written, g read, moments read and
// written), 4 more for the norm. 35 million fp32 parameters: the norm 44 us (3.2 TB/s; twice the workgroups or twice
// the loads in flight gained nothing), 32-bit moments 170 us (5.8 TB/s), 8-bit ones 100 to 112 us by the state (5.6 to
// 5.0 TB/s). Ten tensors of 198 thousand: 9 us, two launches. The tensors' pointers travel as kernel arguments (no
// table in device memory, so a captured step holds what it needs), ADAMW_TENSORS a launch.
#include <cmath>

#include "adamw.h"
#include "fp8_device.h"
#include "rng.h"
#include "siren_common.h"

namespace siren {

namespace {

constexpr int CHUNK = 2048;       // elements of one tensor that a workgroup takes at a time: 16 scale blocks
constexpr int NORM_THREADS = 512;
constexpr int KEY_THREAD = 128;   // where each tensor has its own bias: behind the threads that make those
static_assert(ADAMW_TENSORS <= KEY_THREAD && KEY_THREAD < NORM_THREADS, "a thread a tensor");

// what the update needs of a number of steps t
struct AdamwBias {
    float step_size, inv_root;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
};
// and of the step's own number and the seed, written by the first launch of a step
struct AdamwScalars {
    AdamwBias bias;
    uint64_t key;  // rng_key(seed, t)
};

struct AdamwTable {
    const void* p[ADAMW_TENSORS];
    const void* g[ADAMW_TENSORS];
    int64_t n[ADAMW_TENSORS];
    uint32_t block[ADAMW_TENSORS];  // the tensor's first 128-element block in the flat moments
    uint32_t first[ADAMW_TENSORS];  // its first chunk in this launch
    uint32_t index[ADAMW_TENSORS];  // its place in the caller's list
    int count;
    uint32_t chunks;
};

// the tensor that holds chunk c: the last whose first chunk is at most c (tensors without elements or gradient are not listed)
__device__ __forceinline__ int find_tensor(const AdamwTable& t, uint32_t c) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= c)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

// four consecutive elements of src at i, however they are aligned; those at or past n are zero
template <typename T>
__device__ __forceinline__ f32x4 load4(const T* src, int64_t i, int64_t n) {
    f32x4 r = {0.f, 0.f, 0.f, 0.f};
    if (i + 4 <= n) {
        const typename Quad<T>::Type v = *(const typename Quad<T>::Type*)(src + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = (float)v[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) r[k] = (float)src[i + k];
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void store4(T* dst, int64_t i, int64_t n, f32x4 v) {
    if (i + 4 <= n) {
        *(typename Quad<T>::Type*)(dst + i) = typename Quad<T>::Type{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) dst[i + k] = (T)v[k];
    }
}

__device__ __forceinline__ AdamwBias bias_of(int64_t t, const AdamwHyper& h) {
    const float root = (float)sqrt(1.0 - pow(h.b2, (double)t));
    return {(float)(h.lr / (1.0 - pow(h.b1, (double)t))), 1.f / root};
}
__device__ __forceinline__ int64_t write_key(int64_t* step, AdamwScalars* out, const AdamwHyper& h) {
    const int64_t t = *step + 1;
    *step = t;
    out->key = rng_key(h.seed, (uint64_t)t);
    return t;
}
__device__ __forceinline__ void write_scalars(int64_t* step, AdamwScalars* out, const AdamwHyper& h) {
    out->bias = bias_of(write_key(step, out, h), h);
}
// A tensor whose gradient is missing now and then has taken fewer steps than the list: its moments have decayed less, and its
// corrections go by its own count. One thread a tensor of the table, the step's key in another wave beside them: two powers in
// 64 bits are 1 us of latency.
__device__ __forceinline__ void write_biases(const AdamwTable& tab, int64_t* counts, AdamwBias* out, const AdamwHyper& h) {
    if ((int)threadIdx.x >= tab.count) return;  // ADAMW_TENSORS threads at most
    const int64_t t = counts[tab.index[threadIdx.x]] + 1;
    counts[tab.index[threadIdx.x]] = t;
    out[threadIdx.x] = bias_of(t, h);
}

// the first launch of a step that takes no norm, and with counts each table's
__global__ void adamw_begin_kernel(int64_t* step, AdamwScalars* out, float* norm, AdamwHyper h) {
    write_scalars(step, out, h);
    *norm = 0.f;
}
__global__ void adamw_begin_each_kernel(AdamwTable tab, int64_t* step, AdamwScalars* out, float* norm, int64_t* counts,
                                        AdamwBias* bias, AdamwHyper h) {
    if (step != nullptr && threadIdx.x == KEY_THREAD) {
        write_key(step, out, h);
        *norm = 0.f;
    }
    write_biases(tab, counts, bias, h);
}

// partial[workgroup] = sum of g^2 over its chunks, in 64 bits: the factor c is then the same to its last bit whatever
// the split, and with it every code. Squares of fp32 values are exact in 64 bits.
template <typename T>
__global__ __launch_bounds__(NORM_THREADS) void adamw_norm_kernel(AdamwTable tab, double* __restrict__ partial,
                                                                  int64_t* step, AdamwScalars* out, int64_t* counts,
                                                                  AdamwBias* bias, AdamwHyper h) {
    if (blockIdx.x == 0 && counts != nullptr) {
        if (step != nullptr && threadIdx.x == KEY_THREAD) write_key(step, out, h);
        write_biases(tab, counts, bias, h);
    } else if (blockIdx.x == 0 && step != nullptr && threadIdx.x == 0) {
        write_scalars(step, out, h);
    }
    // four chunks' loads before the first is squared
    double acc = 0.0;
    for (uint32_t c0 = blockIdx.x; c0 < tab.chunks; c0 += 4 * gridDim.x) {
        f32x4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t c = c0 + u * gridDim.x;
            v[u] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (c < tab.chunks) {
                const int k = find_tensor(tab, c);
                v[u] = load4((const T*)tab.g[k], (int64_t)(c - tab.first[k]) * CHUNK + threadIdx.x * 4, tab.n[k]);
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc = fma((double)v[u][e], (double)v[u][e], acc);
    }
    __shared__ double red[NORM_THREADS / 64];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) acc += __shfl_xor(acc, off);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        double s = 0.0;
        for (int w = 0; w < NORM_THREADS / 64; ++w) s += red[w];
        partial[blockIdx.x] = s;
    }
}

// the clip factor from all partial sums, in a fixed order, and the norm for the caller
__device__ __forceinline__ float clip_factor(const double* __restrict__ partial, int parts, double max_norm,
                                             float* __restrict__ norm_out, double* red) {
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += 256) s += partial[i];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3]));
    if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const double c = max_norm / (norm + 1e-6);
    return c > 1.0 ? 1.f : (float)c;  // a NaN norm stays NaN
}

// one element's moments; every operation rounds by itself (no contraction), so that the codes of the 8-bit moments
// do not depend on how a compiler fuses
__device__ __forceinline__ void moments(float g, float& m, float& v, float omb1, float b2, float omb2) {
#pragma clang fp contract(off)
    m = m + (g - m) * omb1;
    v = v * b2 + (g * g) * omb2;
}

// p (1 - lr wd) - step m / (u / root + eps); a reciprocal of one unit in the last place: the update's own error is far
// below p's rounding. u comes from the full square root: the card's own takes a subnormal v for zero, and with a small eps
// the step would be infinite.
__device__ __forceinline__ float apply(float p, float m, float u, float decay, float step_size, float inv_root,
                                       float eps) {
    return __builtin_fmaf(-step_size * m, __builtin_amdgcn_rcpf(__builtin_fmaf(u, inv_root, eps)), p * decay);
}

// A workgroup's first chunk is asked for before the clip factor is made of the partial sums (one round trip less; the 8-bit
// kernel's registers would lose a workgroup a CU for it).
template <typename T, bool EACH>
__global__ __launch_bounds__(256) void adamw32_kernel(AdamwTable tab, float* __restrict__ em, float* __restrict__ ev,
                                                      const AdamwBias* __restrict__ bias, AdamwHyper h,
                                                      const double* __restrict__ partial, int parts,
                                                      float* __restrict__ norm_out) {
    __shared__ double red[4];
    float c = 1.f;
    const AdamwBias all = *bias;
    for (uint32_t ch = blockIdx.x; ch < tab.chunks; ch += gridDim.x) {
        const int k = find_tensor(tab, ch);
        T* p = (T*)tab.p[k];
        const T* g = (const T*)tab.g[k];
        const int64_t n = tab.n[k], off = (int64_t)tab.block[k] * 128;
        const AdamwBias own = EACH ? bias[k] : all;
        const int64_t base = (int64_t)(ch - tab.first[k]) * CHUNK + threadIdx.x * 4;
        f32x4 pv[2], gv[2], mv[2], vv[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int64_t i = base + q * (CHUNK / 2);
            if (i >= n) continue;
            pv[q] = load4(p, i, n);
            gv[q] = load4(g, i, n);
            mv[q] = *(const f32x4*)(em + off + i);  // the pad behind a tensor's end may be read, never written
            vv[q] = *(const f32x4*)(ev + off + i);
        }
        if (ch == blockIdx.x && parts > 0) c = clip_factor(partial, parts, h.max_norm, norm_out, red);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int64_t i = base + q * (CHUNK / 2);
            if (i >= n) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float m = mv[q][e], v = vv[q][e];
                moments(c * gv[q][e], m, v, h.omb1, h.b2f, h.omb2);
                mv[q][e] = m;
                vv[q][e] = v;
                pv[q][e] = apply(pv[q][e], m, __builtin_sqrtf(v), h.decay, own.step_size, own.inv_root, h.epsf);
            }
            store4(p, i, n, pv[q]);
            store4(em + off, i, n, mv[q]);
            store4(ev + off, i, n, vv[q]);
        }
    }
}

// e4m3's code of |x| / scale, rounded up where the 16 bits r say so: the scaled magnitude times 2^-120 is an fp32
// number whose upper 12 bits are the code, subnormal codes among them
__device__ __forceinline__ uint32_t random_code(float x, float inv, uint32_t r) {
#pragma clang fp contract(off)
    const float y = (__builtin_fabsf(x) * inv) * 0x1p-120f;
    return (__float_as_uint(y) + (r << 4)) >> 20;
}

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }

template <typename T, bool EACH>
__global__ __launch_bounds__(256) void adamw8_kernel(AdamwTable tab, uint8_t* __restrict__ em, uint8_t* __restrict__ eu,
                                                     uint8_t* __restrict__ sm, uint8_t* __restrict__ su,
                                                     const AdamwScalars* __restrict__ sc,
                                                     const AdamwBias* __restrict__ bias, AdamwHyper h,
                                                     const double* __restrict__ partial, int parts,
                                                     float* __restrict__ norm_out) {
    __shared__ double red[4];
    const float c = parts > 0 ? clip_factor(partial, parts, h.max_norm, norm_out, red) : 1.f;
    const uint64_t key = sc->key;
    const AdamwBias all = *bias;
    for (uint32_t ch = blockIdx.x; ch < tab.chunks; ch += gridDim.x) {
        const int k = find_tensor(tab, ch);
        T* p = (T*)tab.p[k];
        const T* g = (const T*)tab.g[k];
        const AdamwBias own = EACH ? bias[k] : all;
        const int64_t n = tab.n[k], off = (int64_t)tab.block[k] * 128;
        // 16 lanes hold one block of 128; a block that begins past the tensor's end does not exist
        const int64_t i = (int64_t)(ch - tab.first[k]) * CHUNK + threadIdx.x * 8;
        if ((i & ~(int64_t)127) >= n) continue;
        const int64_t blk = (off + i) >> 7;
        const u32x2 mc = *(const u32x2*)(em + off + i), uc = *(const u32x2*)(eu + off + i);
        const uint8_t msb = sm[blk], usb = su[blk];
        f32x4 pv[2], gv[2];
        if (i + 8 <= n) {  // one branch for all four quads
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                pv[q] = load4(p, i + 4 * q, i + 8);
                gv[q] = load4(g, i + 4 * q, i + 8);
            }
        } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                pv[q] = load4(p, i + 4 * q, n);
                gv[q] = load4(g, i + 4 * q, n);
            }
        }
        const float ms = scale_of(msb), us = scale_of(usb);
        float m[8], u[8];
        float mmax = 0.f, umax = 0.f;
        bool mok = true, uok = true;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x2 md = (q & 1) ? __builtin_amdgcn_cvt_pk_f32_fp8(mc[q >> 1], true)
                                     : __builtin_amdgcn_cvt_pk_f32_fp8(mc[q >> 1], false);
            const f32x2 ud = (q & 1) ? __builtin_amdgcn_cvt_pk_f32_fp8(uc[q >> 1], true)
                                     : __builtin_amdgcn_cvt_pk_f32_fp8(uc[q >> 1], false);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int j = 2 * q + e;
                float mj = md[e] * ms, uj = ud[e] * us;
                float vj = uj * uj;
                moments(c * gv[j >> 2][j & 3], mj, vj, h.omb1, h.b2f, h.omb2);
                uj = __builtin_sqrtf(vj);
                m[j] = mj;
                u[j] = uj;
                mok = mok && finite(mj);
                uok = uok && finite(uj);
                mmax = fmaxf(mmax, __builtin_fabsf(mj));
                umax = fmaxf(umax, uj);
                pv[j >> 2][j & 3] = apply(pv[j >> 2][j & 3], mj, uj, h.decay, own.step_size, own.inv_root, h.epsf);
            }
        }
        // a block with an infinity or a NaN is held as a NaN (byte 255, codes 0); the maximum carries the fact
        mmax = row16_max(mok ? mmax : INFINITY);
        umax = row16_max(uok ? umax : INFINITY);
        const bool mbad = !finite(mmax), ubad = !finite(umax);
        const int mb = exponent_byte<false>(mmax), ub = exponent_byte<false>(umax);
        const float mi = scale_of(254 - mb), ui = scale_of(254 - ub);
        u32x2 mo = {0u, 0u}, uo = {0u, 0u};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint64_t rnd = mix64(key + (uint64_t)((off + i) / 2 + q));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int j = 2 * q + e;
                const uint32_t r = (uint32_t)(rnd >> (32 * e));
                uint32_t cm = random_code(m[j], mi, r & 0xFFFFu) | (m[j] < 0.f ? 0x80u : 0u);
                uint32_t cu = random_code(u[j], ui, r >> 16);
                if (u[j] > 0.f && cu == 0u) cu = 1u;  // a second moment that is not zero is not held as zero
                mo[j >> 2] |= (mbad ? 0u : cm) << (8 * (j & 3));
                uo[j >> 2] |= (ubad ? 0u : cu) << (8 * (j & 3));
            }
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) store4(p, i + 4 * q, n, pv[q]);
        *(u32x2*)(em + off + i) = mo;
        *(u32x2*)(eu + off + i) = uo;
        if ((threadIdx.x & 15) == 0) {
            sm[blk] = (uint8_t)(mbad ? 255 : mb);
            su[blk] = (uint8_t)(ubad ? 255 : ub);
        }
    }
}

}  // namespace

// one table per ADAMW_TENSORS tensors and at most one partly filled per type
static int64_t adamw_tables(int64_t count) { return count / ADAMW_TENSORS + 3; }
int64_t adamw_scratch_bytes(int64_t count) {
    return 64 + adamw_tables(count) * ADAMW_NORM_BLOCKS * (int64_t)sizeof(double) +
           (count * (int64_t)sizeof(AdamwBias) + 15) / 16 * 16;
}

void launch_adamw(hipStream_t st, const AdamwCall& a) {
    // scratch: [scalars][norm, at 32][partial sums, at 64][each listed tensor's bias, in the order of the tables]
    AdamwScalars* sc = (AdamwScalars*)a.scratch;
    float* norm = (float*)((char*)a.scratch + 32);
    double* partial = (double*)((char*)a.scratch + 64);
    AdamwBias* biases = (AdamwBias*)(partial + adamw_tables(a.count) * ADAMW_NORM_BLOCKS);
    const bool each = a.counts != nullptr;
    AdamwTable tab;
    int parts = 0;
    bool begun = false;
    // pass 0: the norm (when clipping) and each tensor's bias (with counts), pass 1: the update. Each walks the tensors type by
    // type, a table at a time.
    for (int pass = a.h.max_norm > 0.0 || each ? 0 : 1; pass < 2; ++pass) {
        if (!begun && pass == 1) {
            hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(1), 0, st, a.step, sc, norm, a.h);
            begun = true;
        }
        int64_t listed = 0;
        for (int type = 0; type < 3; ++type) {
            tab.count = 0;
            tab.chunks = 0;
            auto flush = [&]() {
                if (tab.count == 0) return;
                AdamwBias* bias = biases + listed;
                listed += tab.count;
                if (pass == 0) {
                    const unsigned grid = tab.chunks < (uint32_t)ADAMW_NORM_BLOCKS ? tab.chunks : ADAMW_NORM_BLOCKS;
                    int64_t* step = begun ? nullptr : a.step;
                    begun = true;
#define SIREN_ADAMW_NORM(T)                                                                                                  \
    hipLaunchKernelGGL(adamw_norm_kernel<T>, dim3(grid), dim3(NORM_THREADS), 0, st, tab, partial + parts, step, sc, a.counts, \
                       bias, a.h)
                    if (!(a.h.max_norm > 0.0)) {
                        hipLaunchKernelGGL(adamw_begin_each_kernel, dim3(1), dim3(KEY_THREAD + 1), 0, st, tab, step, sc, norm, a.counts, bias,
                                           a.h);
                    } else {
                        if (type == 0) SIREN_ADAMW_NORM(float);
                        if (type == 1) SIREN_ADAMW_NORM(__bf16);
                        if (type == 2) SIREN_ADAMW_NORM(_Float16);
                        parts += (int)grid;
                    }
#undef SIREN_ADAMW_NORM
                } else {
                    const unsigned grid = tab.chunks < (uint32_t)ADAMW_BLOCKS ? tab.chunks : ADAMW_BLOCKS;
                    if (!each) bias = &sc->bias;
#define SIREN_ADAMW(T, EACH)                                                                                                   \
    do {                                                                                                                       \
        if (a.bits == 32)                                                                                                      \
            hipLaunchKernelGGL((adamw32_kernel<T, EACH>), dim3(grid), dim3(256), 0, st, tab, (float*)a.m, (float*)a.v, bias,   \
                               a.h, partial, parts, norm);                                                                     \
        else                                                                                                                   \
            hipLaunchKernelGGL((adamw8_kernel<T, EACH>), dim3(grid), dim3(256), 0, st, tab, (uint8_t*)a.m, (uint8_t*)a.v,      \
                               a.sm, a.sv, sc, bias, a.h, partial, parts, norm);                                               \
    } while (0)
#define SIREN_ADAMW_TYPES(EACH)                 \
    do {                                        \
        if (type == 0) SIREN_ADAMW(float, EACH);    \
        if (type == 1) SIREN_ADAMW(__bf16, EACH);   \
        if (type == 2) SIREN_ADAMW(_Float16, EACH); \
    } while (0)
                    if (each)
                        SIREN_ADAMW_TYPES(true);
                    else
                        SIREN_ADAMW_TYPES(false);
#undef SIREN_ADAMW_TYPES
#undef SIREN_ADAMW
                }
                tab.count = 0;
                tab.chunks = 0;
            };
            int64_t block = 0;
            for (int64_t k = 0; k < a.count; ++k) {
                const int64_t n = a.numel[k];
                if (a.dtype[k] == type && n > 0 && a.g[k] != nullptr) {
                    const int64_t chunks = (n + CHUNK - 1) / CHUNK;
                    if (tab.count == ADAMW_TENSORS || tab.chunks + chunks > 0x7FFFFFFF) flush();
                    tab.p[tab.count] = a.p[k];
                    tab.g[tab.count] = a.g[k];
                    tab.n[tab.count] = n;
                    tab.block[tab.count] = (uint32_t)block;
                    tab.first[tab.count] = tab.chunks;
                    tab.index[tab.count] = (uint32_t)k;
                    tab.chunks += (uint32_t)chunks;
                    ++tab.count;
                }
                block += (n + 127) / 128;
            }
            flush();
        }
    }
}

}  // namespace siren
