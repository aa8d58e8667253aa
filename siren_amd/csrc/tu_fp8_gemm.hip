// tu_fp8_gemm.hip — the product of two 8-bit operands with block scales: out = act(A B^T + bias).
//
//   out[m][n] = sum_b sa[m][b] sb[n][b] sum_{k in block b} a[m][k] b[n][k], 32-bit sums
//
// The card's fp8 matrix instructions keep about 17 bits of the products that one instruction sums (errors of 1e-5 of
// the result on random operands, whatever the length), the bf16 ones lose nothing of these operands' products; an e4m3
// value times a power of two is a bf16 number exactly, and v_cvt_scalef32_pk_bf16_fp8 makes two of them at once. So the
// operands travel as bytes through HBM and LDS, are scaled and widened in registers, and the bf16 matrix pipe sums them.
//
// A workgroup of 4 waves owns 128 x 128 of out, each wave 64 x 64 (16 accumulators of 16 x 16). A step takes one block
// of 128 k of both operands: 16 + 16 KiB by direct global-to-LDS loads, two buffers, so one step's loads run behind the
// other's products. An LDS row is the 128 bytes of one operand row; its 16-byte pieces are permuted by (row >> 1) & 7 on
// the way in, so that the 16 lanes that read one piece of 16 rows hit distinct banks. The sums do not care in which
// order k is taken as long as both operands agree: piece p of a row serves as k-slices 2p, 2p + 1 of 8 x 8.
#include "fp8.h"
#include "siren_common.h"

namespace siren {

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int TM = 128, TN = 128, BK = 128;  // workgroup tile, k of one step
constexpr int OPERAND = 128 * BK;            // bytes of one operand's step

struct GemmArgs {
    const uint8_t *a, *b, *sa, *sb;
    int64_t lda, ldb, lsa, lsb;  // bytes of a row, of a row's scales
    int64_t m, n;
    int sha, shb;                // scales per row (0) or per 128 rows (7)
    int steps, steps_per_split;  // blocks of k, and of one split
    int tiles_m, tiles_n;
    const float* bias;
    int act;
    float omega;
    void* out;                   // split: fp32 partial products (splits, m, n)
    __bf16* deriv;
};

template <bool E5M2, int HI>
__device__ __forceinline__ bf16x2 widen2(uint32_t w, float scale) {
    if constexpr (E5M2)
        return __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, scale, HI);
    else
        return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI);
}
// 8 bytes (two words) -> 8 bf16 numbers, times scale
template <bool E5M2>
__device__ __forceinline__ bf16x8 widen8(uint32_t w0, uint32_t w1, float scale) {
    const bf16x2 p0 = widen2<E5M2, 0>(w0, scale), p1 = widen2<E5M2, 1>(w0, scale);
    const bf16x2 p2 = widen2<E5M2, 0>(w1, scale), p3 = widen2<E5M2, 1>(w1, scale);
    return bf16x8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}

template <typename T>
__device__ __forceinline__ void put4(T* dst, f32x4 v, int valid, bool vec) {
    if (vec && valid >= 4) {
        if constexpr (sizeof(T) == 4) {
            *(f32x4*)dst = v;
        } else {
            typedef T T4 __attribute__((ext_vector_type(4)));
            *(T4*)dst = T4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < valid) dst[k] = (T)v[k];
    }
}

// bias, sine and the store of out[row][col .. col + 3]
template <typename T>
__device__ __forceinline__ void finish(const GemmArgs& g, int64_t row, int64_t col, f32x4 v) {
    const int64_t left = g.n - col;
    const int valid = left < 4 ? (int)left : 4;
    const bool vec = (g.n & 3) == 0;
    if (g.bias != nullptr) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < valid) v[k] += g.bias[col + k];
    }
    if (g.act == FP8_ACT_SINE) {
        f32x4 t = v * g.omega;
        const float top = fmaxf(fmaxf(__builtin_fabsf(t[0]), __builtin_fabsf(t[1])),
                                fmaxf(__builtin_fabsf(t[2]), __builtin_fabsf(t[3])));
        if (__builtin_expect(top > 1.0e5f, 0)) {  // past the reduction's exact range
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = sinf(t[k]);
            if (g.deriv != nullptr) {
#pragma unroll
                for (int k = 0; k < 4; ++k) t[k] = g.omega * cosf(t[k]);
                put4(g.deriv + row * g.n + col, t, valid, vec);
            }
        } else {
            f32x4 d;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float sn, cs;
                sincos_fast(t[k], sn, cs);  // 4e-7; the cosine falls away where nothing takes it
                v[k] = sn;
                d[k] = g.omega * cs;
            }
            if (g.deriv != nullptr) put4(g.deriv + row * g.n + col, d, valid, vec);
        }
    }
    put4((T*)g.out + row * g.n + col, v, valid, vec);
}

template <typename T, bool E5M2A, bool SPLIT>
__global__ __launch_bounds__(256, 2) void gemm_kernel(GemmArgs g) {
    __shared__ __align__(16) uint8_t lds[2][2][OPERAND];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int r = lane & 15, q = lane >> 4;
    const int wm = wave & 1, wn = wave >> 1;

    // workgroups go round-robin to the 8 dies: give each die a contiguous run of tiles, columns fastest, so that the
    // tiles that share rows of A meet in one L2
    const int tiles = g.tiles_m * g.tiles_n;
    int tile = blockIdx.x;
    {
        const int per = tiles / 8, rest = tiles % 8, x = tile & 7, y = tile >> 3;
        tile = x * per + (x < rest ? x : rest) + y;
    }
    const int64_t m0 = (int64_t)(tile / g.tiles_n) * TM, n0 = (int64_t)(tile % g.tiles_n) * TN;
    const int first = blockIdx.y * g.steps_per_split;
    const int last = first + g.steps_per_split < g.steps ? first + g.steps_per_split : g.steps;

    // this thread's pieces of a step: rows (wave * 4 + j) * 8 + lane / 8, piece lane % 8 of the permuted row. Rows past
    // the operand's end read its last row; their products are not stored.
    const uint8_t *pa[4], *pb[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int row = (wave * 4 + j) * 8 + (lane >> 3);
        const int piece = (lane & 7) ^ ((row >> 1) & 7);
        const int64_t ra = m0 + row < g.m ? m0 + row : g.m - 1, rb = n0 + row < g.n ? n0 + row : g.n - 1;
        pa[j] = g.a + ra * g.lda + (int64_t)first * BK + piece * 16;
        pb[j] = g.b + rb * g.ldb + (int64_t)first * BK + piece * 16;
    }
    auto load = [&](int buf) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)pa[j],
                                             (__attribute__((address_space(3))) void*)(lds[buf][0] + (wave * 4 + j) * 1024),
                                             16, 0, 0);
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)pb[j],
                                             (__attribute__((address_space(3))) void*)(lds[buf][1] + (wave * 4 + j) * 1024),
                                             16, 0, 0);
            pa[j] += BK;
            pb[j] += BK;
        }
    };

    // the scales of this lane's rows, four steps to a word
    const uint8_t *qa[4], *qb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t ra = m0 + wm * 64 + i * 16 + r, rb = n0 + wn * 64 + i * 16 + r;
        qa[i] = g.sa + ((ra < g.m ? ra : g.m - 1) >> g.sha) * g.lsa;
        qb[i] = g.sb + ((rb < g.n ? rb : g.n - 1) >> g.shb) * g.lsb;
    }

    f32x4 acc[4][4] = {};
    uint32_t wa[4], wb[4];
    load(0);
    for (int step = first; step < last; ++step) {
        const int buf = (step - first) & 1;
        if (step == first || (step & 3) == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                wa[i] = *(const uint32_t*)(qa[i] + (step & ~3));
                wb[i] = *(const uint32_t*)(qb[i] + (step & ~3));
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's direct-to-LDS loads of this step
        __syncthreads();  // every wave's are in, and the other buffer has been read
        if (step + 1 < last) load(buf ^ 1);
        const int shift = 8 * (step & 3);
        float fa[4], fb[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            fa[i] = __uint_as_float(((wa[i] >> shift) & 0xFFu) << 23);
            fb[i] = __uint_as_float(((wb[i] >> shift) & 0xFFu) << 23);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = r * BK + (((h * 4 + q) ^ ((r >> 1) & 7)) * 16);
            bf16x8 va[4][2], vb[4][2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const u32x4 ba = *(const u32x4*)(lds[buf][0] + (wm * 64 + i * 16) * BK + at);
                const u32x4 bb = *(const u32x4*)(lds[buf][1] + (wn * 64 + i * 16) * BK + at);
                va[i][0] = widen8<E5M2A>(ba[0], ba[1], fa[i]);
                va[i][1] = widen8<E5M2A>(ba[2], ba[3], fa[i]);
                vb[i][0] = widen8<false>(bb[0], bb[1], fb[i]);
                vb[i][1] = widen8<false>(bb[2], bb[3], fb[i]);
            }
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb[j][p], va[i][p], acc[i][j], 0, 0, 0);
        }
    }

    // B rows are the instruction's rows: lane (r, q) holds out[m][n .. n + 3] with m = r, n = 4 q of each 16 x 16
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = m0 + wm * 64 + i * 16 + r;
        if (row >= g.m) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t col = n0 + wn * 64 + j * 16 + q * 4;
            if (col >= g.n) continue;
            if constexpr (SPLIT) {
                const int64_t left = g.n - col;
                put4((float*)g.out + ((int64_t)blockIdx.y * g.m + row) * g.n + col, acc[i][j],
                     left < 4 ? (int)left : 4, (g.n & 3) == 0);
            } else {
                finish<T>(g, row, col, acc[i][j]);
            }
        }
    }
}

// out = act(sum of the splits' partial products + bias), four columns a thread. GROUPS threads share an element's splits,
// each its own contiguous run of them, and are added in order: few outputs with many splits (a reduction over 65536)
// would otherwise leave most of the card idle behind one long chain of loads (33 us for 32 x 256 of 128 splits).
template <typename T, int GROUPS>
__global__ __launch_bounds__(256) void join_kernel(GemmArgs g, const float* __restrict__ part, int splits) {
    constexpr int QUADS = 256 / GROUPS;
    __shared__ f32x4 red[GROUPS][QUADS];
    const int64_t n4 = (g.n + 3) / 4, total = g.m * n4, plane = g.m * g.n;
    const int grp = threadIdx.x / QUADS, at = threadIdx.x % QUADS;
    const int per = (splits + GROUPS - 1) / GROUPS;
    const int lo = grp * per, hi = lo + per < splits ? lo + per : splits;
    for (int64_t base = (int64_t)blockIdx.x * QUADS; base < total; base += (int64_t)gridDim.x * QUADS) {
        const int64_t i = base + at;
        const int64_t row = i / n4, col = (i - row * n4) * 4;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (i < total) {
            const float* src = part + row * g.n + col;
            if ((g.n & 3) == 0) {
#pragma unroll 8
                for (int s = lo; s < hi; ++s) v += *(const f32x4*)(src + s * plane);
            } else {
                for (int s = lo; s < hi; ++s)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (col + k < g.n) v[k] += src[s * plane + k];
            }
        }
        if (GROUPS > 1) {
            red[grp][at] = v;
            __syncthreads();
            if (grp == 0) {
#pragma unroll
                for (int k = 1; k < GROUPS; ++k) v += red[k][at];
            }
            __syncthreads();
        }
        if (grp == 0 && i < total) finish<T>(g, row, col, v);
    }
}

template <typename T>
void launch_join(hipStream_t stream, const GemmArgs& g, const void* part, int splits) {
    const int64_t quads = g.m * ((g.n + 3) / 4);
    // 8 waves a CU of one thread an element is 131072 elements; below that, threads share them
    const bool share = quads < 131072 && splits >= 16;
    const int64_t want = share ? (quads + 15) / 16 : (quads + 255) / 256;
    const dim3 grid((unsigned)(want < 8192 ? want : 8192));
    if (share)
        hipLaunchKernelGGL((join_kernel<T, 16>), grid, dim3(256), 0, stream, g, (const float*)part, splits);
    else
        hipLaunchKernelGGL((join_kernel<T, 1>), grid, dim3(256), 0, stream, g, (const float*)part, splits);
}

// splits of the k axis: enough workgroups to fill 256 CUs twice, at least 4 steps each
int splits_of(int64_t m, int64_t n, int64_t k) {
    const int64_t tiles = ((m + TM - 1) / TM) * ((n + TN - 1) / TN), steps = fp8_blocks(k);
    if (tiles >= 256 || steps < 8) return 1;
    int64_t s = (512 + tiles - 1) / tiles;
    if (s > steps / 4) s = steps / 4;
    const int64_t per = (steps + s - 1) / s;
    return (int)((steps + per - 1) / per);
}

}  // namespace

int64_t fp8_product_ws_bytes(int64_t m, int64_t n, int64_t k) {
    const int s = splits_of(m, n, k);
    return s > 1 ? (int64_t)s * m * n * 4 : 0;
}

void launch_fp8_product(hipStream_t stream, const Fp8Product& p) {
    GemmArgs g;
    g.a = p.a.data;
    g.b = p.b.data;
    g.sa = p.a.scale;
    g.sb = p.b.scale;
    g.lda = g.ldb = fp8_padded(p.k);
    g.lsa = g.lsb = fp8_scale_cols(p.k);
    g.m = p.a.rows;
    g.n = p.b.rows;
    g.sha = p.a.shift;
    g.shb = p.b.shift;
    g.steps = (int)fp8_blocks(p.k);
    g.tiles_m = (int)((g.m + TM - 1) / TM);
    g.tiles_n = (int)((g.n + TN - 1) / TN);
    g.bias = p.bias;
    g.act = p.act;
    g.omega = p.omega;
    g.deriv = (__bf16*)p.deriv;
    const int splits = splits_of(g.m, g.n, p.k);
    g.steps_per_split = (g.steps + splits - 1) / splits;
    g.out = splits > 1 ? p.ws : p.out;
    const dim3 grid((unsigned)(g.tiles_m * g.tiles_n), (unsigned)splits);
#define SIREN_GEMM(T, E, S) hipLaunchKernelGGL((gemm_kernel<T, E, S>), grid, dim3(256), 0, stream, g)
    if (splits > 1) {
        if (p.e5m2_a)
            SIREN_GEMM(float, true, true);
        else
            SIREN_GEMM(float, false, true);
        g.out = p.out;
        if (p.type == FP8_F32) launch_join<float>(stream, g, p.ws, splits);
        if (p.type == FP8_BF16) launch_join<__bf16>(stream, g, p.ws, splits);
        if (p.type == FP8_F16) launch_join<_Float16>(stream, g, p.ws, splits);
        return;
    }
    if (p.e5m2_a) {
        if (p.type == FP8_F32) SIREN_GEMM(float, true, false);
        if (p.type == FP8_BF16) SIREN_GEMM(__bf16, true, false);
        if (p.type == FP8_F16) SIREN_GEMM(_Float16, true, false);
    } else {
        if (p.type == FP8_F32) SIREN_GEMM(float, false, false);
        if (p.type == FP8_BF16) SIREN_GEMM(__bf16, false, false);
        if (p.type == FP8_F16) SIREN_GEMM(_Float16, false, false);
    }
#undef SIREN_GEMM
}

}  // namespace siren
