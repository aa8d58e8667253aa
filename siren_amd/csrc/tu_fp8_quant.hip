// tu_fp8_quant.hip — rounding tensors to 8 bits with a scale for each block of 128.
//
//   s = 2^e, the smallest with which the block's largest finite magnitude is at most 448 s (e5m2: 57344 s), e >= -126
//   q = x / s to the nearest e4m3 (e5m2) value, ties to even; infinities and NaN become NaN (e5m2 keeps infinities)
//
// A power of two divides exactly, so the one rounding is q's, and a dequantised value is a bf16 number exactly (from 2^-133 to
// below 2^128: what of the smallest and largest blocks lies beyond is said with the products).
// A training step needs a tensor both as rows (blocks along the columns) and transposed (blocks along the rows, for
// the product that sums over the rows): one workgroup holds a 128 x 128 tile in registers and writes both, with the
// column sums of a bias's gradient on the way, so the tensor is read once. 64 values a thread: 16 rows x 4 columns, so
// a row's maximum is a reduction over half a wave, a column's one over LDS, and the transpose leaves as 16-byte pieces.
// Bytes bound it: 262144 x 1024 fp32 into both layouts 301 us (1.6 GB, 5.3 TB/s), bf16 214 us (5.0 TB/s; a bf16 value costs
// the same instructions for half the bytes); rows alone 225 us from fp32 (6.0 TB/s).
#include "fp8.h"
#include "fp8_device.h"
#include "siren_common.h"

namespace siren {

namespace {

constexpr int QT = 128;           // tile edge
constexpr int QSTRIDE = QT + 16;  // LDS row of the transposed bytes: 16-byte pieces on distinct banks

struct QuantArgs {
    const void* x;
    int64_t ld, rows, cols;
    const __bf16* mult;
    uint8_t *q, *s, *qt, *st;
    float* colsum;
    int tiles, near, col_blocks, panels;
};

// One tensor, or two in one launch (a layer's x and weight: small ones are all launch): workgroups from `first` on take b's
// tiles.
template <typename T, bool E5M2, bool MULT>
__global__ __launch_bounds__(256, 4) void quant_kernel(QuantArgs a, QuantArgs b, unsigned first) {
    const bool second = blockIdx.x >= first;
    const QuantArgs& arg = second ? b : a;
    const unsigned tile = second ? blockIdx.x - first : blockIdx.x;
    const T* __restrict__ x = (const T*)arg.x;
    const int64_t ld = arg.ld, rows = arg.rows, cols = arg.cols;
    const __bf16* __restrict__ mult = arg.mult;
    uint8_t* __restrict__ q = arg.q;
    uint8_t* __restrict__ s = arg.s;
    uint8_t* __restrict__ qt = arg.qt;
    uint8_t* __restrict__ st = arg.st;
    float* __restrict__ colsum = arg.colsum;
    const int tiles = arg.tiles, near = arg.near, col_blocks = arg.col_blocks, panels = arg.panels;
    __shared__ __align__(16) uint8_t tr[QT * QSTRIDE];
    __shared__ float part[8][QT];
    __shared__ float wmax[4];
    const int t = threadIdx.x, c4 = t & 31, rg = t >> 5;
    const int64_t rb = tile / (unsigned)col_blocks;
    const int cb = (int)(tile % (unsigned)col_blocks);
    const int64_t r0 = rb * QT + rg * 16;
    const int64_t c0 = (int64_t)cb * QT + c4 * 4;
    const int64_t row_blocks = (rows + QT - 1) / QT;
    const int64_t s_ld = (col_blocks + 3) / 4 * 4, st_ld = (row_blocks + 3) / 4 * 4;

    // Every load is issued before any is waited for (a branch around each row's load made 16 round trips of them: 8 us for
    // one row), by the wave's uniform address and a 32-bit offset of the lane (64-bit addresses of 16 rows cost the fourth
    // wave of a SIMD). A tile on the edge reads the last row again, and columns up to the last, and zeroes what does not exist.
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int64_t wr = rb * QT + wave * 32;  // the wave's first row
    f32x4 v[16];
    typedef typename Quad<T>::Type T4;
    typedef typename Quad<__bf16>::Type B4;
    if (near && (rb + 1) * QT <= rows && (int64_t)(cb + 1) * QT <= cols) {
        const uint32_t row = (rg & 1) * 16, at = (row * (uint32_t)ld + c4 * 4) * (uint32_t)sizeof(T);
        const T* src = x + wr * ld + (int64_t)cb * QT;
        T4 h[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) h[i] = *(const T4*)((const char*)(src + i * ld) + at);
        if constexpr (MULT) {
            const uint32_t mat = (row * (uint32_t)cols + c4 * 4) * 2u;
            const __bf16* msrc = mult + wr * cols + (int64_t)cb * QT;
            B4 f[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) f[i] = *(const B4*)((const char*)(msrc + i * cols) + mat);
#pragma unroll
            for (int i = 0; i < 16; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) v[i][k] = (float)h[i][k] * (float)f[i][k];
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) v[i][k] = (float)h[i][k];
        }
    } else if (wr >= rows) {  // nothing of this wave's rows exists
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    } else if (near && cols >= 4) {
        // the quad that crosses the end is read up to the end and shifted
        const int64_t cs = c0 < cols - 4 ? c0 : cols - 4;
        const int shift = c0 - cs < 4 ? (int)(c0 - cs) : 4, left = (int)(rows - 1 - wr < 31 ? rows - 1 - wr : 31);
        const T* src = x + wr * ld + (int64_t)cb * QT;
        const __bf16* msrc = mult + wr * cols + (int64_t)cb * QT;
        const int c = (int)(cs - (int64_t)cb * QT);  // may be negative: the address below is taken in 64 bits then
        T4 h[16];
        B4 f[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int r = (rg & 1) * 16 + i < left ? (rg & 1) * 16 + i : left;
            h[i] = *(const T4*)((const char*)(src + c) + (uint32_t)r * (uint32_t)ld * (uint32_t)sizeof(T));
            if constexpr (MULT) f[i] = *(const B4*)((const char*)(msrc + c) + (uint32_t)r * (uint32_t)cols * 2u);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float p[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                p[k] = (float)h[i][k];
                if constexpr (MULT) p[k] *= (float)f[i][k];
            }
            const bool in = r0 + i < rows;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[i][k] = in ? p[k] : 0.f;
        }
        if ((int64_t)(cb + 1) * QT > cols) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const f32x4 p = v[i];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float u = shift == 0 ? p[k] : 0.f;
#pragma unroll
                    for (int d = 1; d < 4 - k; ++d) u = shift == d ? p[k + d] : u;
                    v[i][k] = u;
                }
            }
        }
    } else {
        // fewer than 4 columns, or rows 2^25 elements apart: four rows at a time
#pragma unroll
        for (int b = 0; b < 4; ++b) {
#pragma unroll
            for (int i = 4 * b; i < 4 * b + 4; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const bool in = r0 + i < rows && c0 + k < cols;
                    v[i][k] = in ? (float)x[(r0 + i) * ld + c0 + k] : 0.f;
                    if (MULT && in) v[i][k] *= (float)mult[(r0 + i) * cols + c0 + k];
                }
            asm volatile("" ::: "memory");
        }
    }

    if (colsum != nullptr) {  // 16 rows a thread, then the 8 row groups in order
        f32x4 sum = v[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) sum += v[i];
#pragma unroll
        for (int k = 0; k < 4; ++k) part[rg][c4 * 4 + k] = sum[k];
        __syncthreads();
        if (t < QT && (int64_t)cb * QT + t < cols) {
            float a = part[0][t];
#pragma unroll
            for (int g = 1; g < 8; ++g) a += part[g][t];
            colsum[rb * cols + (int64_t)cb * QT + t] = a;
        }
        __syncthreads();
    }

    int tile_byte = 0;
    if (tiles) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) m = fmaxf(m, __builtin_fabsf(v[i][k]));
        if (__builtin_expect(__any(m == INFINITY), 0)) {  // fmaxf drops NaN; infinities are dropped here
            m = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) m = fmaxf(m, finite_abs(v[i][k]));
        }
        m = half_wave_max(m);
        m = fmaxf(m, __shfl_xor(m, 32));
        if ((t & 63) == 0) wmax[t >> 6] = m;
        __syncthreads();
        tile_byte = exponent_byte<E5M2>(fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3])));
        // pad bytes of the last word stand for 1
        if (s != nullptr && t == 0) {
            s[rb * s_ld + cb] = (uint8_t)tile_byte;
            if (cb == col_blocks - 1)
                for (int64_t p = col_blocks; p < s_ld; ++p) s[rb * s_ld + p] = 127;
        }
        if (st != nullptr && t == 0) {
            st[(int64_t)cb * st_ld + rb] = (uint8_t)tile_byte;
            if (rb == row_blocks - 1)
                for (int64_t p = row_blocks; p < st_ld; ++p) st[(int64_t)cb * st_ld + p] = 127;
        }
    }

    if (q != nullptr) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            int byte = tile_byte;
            if (!tiles) byte = exponent_byte<E5M2>(half_wave_amax(v[i][0], v[i][1], v[i][2], v[i][3]));
            if (r0 + i < rows) {
                uint8_t* dst = (panels & 1) ? q + ((cb * 2 + (c4 >> 4)) * rows + r0 + i) * 64 + (c4 & 15) * 4
                                      : q + (r0 + i) * ((int64_t)col_blocks * QT) + c0;
                *(uint32_t*)dst =
                    pack4<E5M2>(v[i][0], v[i][1], v[i][2], v[i][3], scale_of(byte));
                if (!tiles && c4 == 0) {
                    s[(r0 + i) * s_ld + cb] = (uint8_t)byte;
                    if (cb == col_blocks - 1)
                        for (int64_t p = col_blocks; p < s_ld; ++p) s[(r0 + i) * s_ld + p] = 127;
                }
            }
        }
    }

    if (qt != nullptr) {
        float scale[4];
        if (tiles) {
#pragma unroll
            for (int k = 0; k < 4; ++k) scale[k] = scale_of(tile_byte);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float m = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) m = fmaxf(m, __builtin_fabsf(v[i][k]));
                if (__builtin_expect(__any(m == INFINITY), 0)) {
                    m = 0.f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) m = fmaxf(m, finite_abs(v[i][k]));
                }
                part[rg][c4 * 4 + k] = m;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float m = part[0][c4 * 4 + k];
#pragma unroll
                for (int g = 1; g < 8; ++g) m = fmaxf(m, part[g][c4 * 4 + k]);
                const int byte = exponent_byte<E5M2>(m);
                scale[k] = scale_of(byte);
                if (rg == 0 && c0 + k < cols) {
                    st[(c0 + k) * st_ld + rb] = (uint8_t)byte;
                    if (rb == row_blocks - 1)
                        for (int64_t p = row_blocks; p < st_ld; ++p) st[(c0 + k) * st_ld + p] = 127;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            u32x4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[j] = pack4<E5M2>(v[4 * j][k], v[4 * j + 1][k], v[4 * j + 2][k], v[4 * j + 3][k], scale[k]);
            *(u32x4*)(tr + (c4 * 4 + k) * QSTRIDE + rg * 16) = w;
        }
        __syncthreads();
        if (panels & 2) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // 4 lanes a column of each panel: a wave's 16 columns lie behind each other
                const int c = (j & 1) * 64 + (t >> 2), piece = (j >> 1) * 4 + (t & 3);
                if ((int64_t)cb * QT + c < cols)  // nontemporal: 262144 x 1024 fp32 313 -> 301 us
                    __builtin_nontemporal_store(*(const u32x4*)(tr + c * QSTRIDE + piece * 16),
                                                (u32x4*)(qt + ((rb * 2 + (j >> 1)) * cols + (int64_t)cb * QT + c) * 64 + (t & 3) * 16));
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // 8 lanes a column: 128 contiguous bytes of the transpose
                const int c = j * 32 + (t >> 3), piece = t & 7;
                if ((int64_t)cb * QT + c < cols)
                    *(u32x4*)(qt + ((int64_t)cb * QT + c) * (row_blocks * QT) + rb * QT + piece * 16) =
                        *(const u32x4*)(tr + c * QSTRIDE + piece * 16);
            }
        }
    }
}

// Rows alone, nothing transposed (a layer that is only evaluated): 16 bytes a lane, so half a wave (a quarter, of 16-bit
// values) takes one block of a row, and a workgroup one block of 32 (64) rows, 4 a unit, all loaded before any is reduced. A few
// rows are a matter of latency here (the tile kernel above is thousands of instructions long, 8 us for one row), many one of
// bytes: 16384 x 1024 bf16 11 us (4.5 TB/s), 262144 x 1024 fp32 226 us (5.9 TB/s).
template <typename T>
constexpr int ROW_LANES = sizeof(T) == 4 ? 32 : 16;
template <typename T>
constexpr int ROWS_PER_GROUP = 4 * 256 / ROW_LANES<T>;
template <typename T, bool E5M2>
__global__ __launch_bounds__(256) void quant_rows_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int64_t cols,
                                                         uint8_t* __restrict__ q, uint8_t* __restrict__ s,
                                                         int col_blocks, int panels) {
    constexpr int LANES = ROW_LANES<T>, QUADS = 32 / LANES, UNITS = 256 / LANES;
    const int lane = threadIdx.x & (LANES - 1), unit = threadIdx.x / LANES;
    const int64_t rb = blockIdx.x / col_blocks;
    const int cb = (int)(blockIdx.x % col_blocks);
    const int col = lane * 4 * QUADS;  // in the block
    const int64_t c0 = (int64_t)cb * QT + col;
    const int64_t s_ld = (col_blocks + 3) / 4 * 4;
    float v[4][QUADS][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = rb * ROWS_PER_GROUP<T> + i * UNITS + unit;
        const T* src = x + (r < rows ? r : rows - 1) * ld + c0;
        if (QUADS == 2 && c0 + 8 <= cols) {
            typedef T Oct __attribute__((ext_vector_type(8), aligned(sizeof(T))));
            const Oct h = *(const Oct*)src;
#pragma unroll
            for (int k = 0; k < 4 * QUADS; ++k) v[i][k >> 2][k & 3] = (float)h[k];
        } else {
#pragma unroll
            for (int d = 0; d < QUADS; ++d) {
                const int64_t left = cols - c0 - 4 * d;
                load_quad(src + 4 * d, left < 4 ? (left > 0 ? (int)left : 0) : 4, v[i][d]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = rb * ROWS_PER_GROUP<T> + i * UNITS + unit;
        const int byte = exponent_byte<E5M2>(block_amax<QUADS>(v[i]));
        if (r < rows) {
            uint32_t* dst = (uint32_t*)((panels & 1) ? q + ((cb * 2 + (col >> 6)) * rows + r) * 64 + (col & 63)
                                                     : q + r * ((int64_t)col_blocks * QT) + c0);
            uint32_t w[QUADS];
#pragma unroll
            for (int d = 0; d < QUADS; ++d) w[d] = pack4<E5M2>(v[i][d][0], v[i][d][1], v[i][d][2], v[i][d][3], scale_of(byte));
            if constexpr (QUADS == 2)
                *(u32x2*)dst = u32x2{w[0], w[1]};
            else
                *dst = w[0];
            // the pad bytes of a row's last word stand for 1
            if (lane == 0) s[r * s_ld + cb] = (uint8_t)byte;
            if (cb == col_blocks - 1 && lane > 0 && cb + lane < s_ld) s[r * s_ld + cb + lane] = 127;
        }
    }
}

// out[c] = sum_b colsum[b][c] in 64 bits: 32 columns x 32 groups of row blocks a workgroup, the groups joined in a fixed
// order (4 groups of 64 columns left 16 workgroups for 1024 columns: 213 us for 2048 row blocks)
__global__ __launch_bounds__(1024) void colsum_kernel(const float* __restrict__ colsum, int64_t blocks, int64_t cols,
                                                      float* __restrict__ out) {
    __shared__ double red[32][33];
    const int t = threadIdx.x & 31, g = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + t;
    double a = 0.0;
    if (c < cols) {
#pragma unroll 8
        for (int64_t b = g; b < blocks; b += 32) a += (double)colsum[b * cols + c];
    }
    red[g][t] = a;
    __syncthreads();
    if (g == 0 && c < cols) {
        for (int k = 1; k < 32; ++k) a += red[k][t];
        out[c] = (float)a;
    }
}

}  // namespace

namespace {

bool rows_only(const Fp8Quant& a) { return a.qt == nullptr && a.colsum == nullptr && a.mult == nullptr && !a.tiles; }

QuantArgs args_of(const Fp8Quant& a) {
    const int near = a.rows == 1 || a.ld < 1 << 25;  // 31 rows are less than 2^32 bytes apart
    return QuantArgs{a.x, a.ld, a.rows, a.cols, (const __bf16*)a.mult, a.q, a.s, a.qt, a.st, a.colsum, a.tiles, near,
                     (int)fp8_blocks(a.cols), a.panels};
}

unsigned tiles_in(const Fp8Quant& a) { return (unsigned)(fp8_blocks(a.rows) * fp8_blocks(a.cols)); }

void launch_tiles(hipStream_t stream, const Fp8Quant& a, const Fp8Quant* b) {
    const QuantArgs first = args_of(a), second = b != nullptr ? args_of(*b) : first;
    const unsigned n = tiles_in(a);
    const dim3 grid(n + (b != nullptr ? tiles_in(*b) : 0u));
#define SIREN_QUANT(T, E, M) hipLaunchKernelGGL((quant_kernel<T, E, M>), grid, dim3(256), 0, stream, first, second, n)
#define SIREN_QUANT_TYPES(E, M)                              \
    do {                                                     \
        if (a.type == FP8_F32) SIREN_QUANT(float, E, M);     \
        if (a.type == FP8_BF16) SIREN_QUANT(__bf16, E, M);   \
        if (a.type == FP8_F16) SIREN_QUANT(_Float16, E, M);  \
    } while (0)
    if (a.e5m2 && a.mult != nullptr)
        SIREN_QUANT_TYPES(true, true);
    else if (a.e5m2)
        SIREN_QUANT_TYPES(true, false);
    else if (a.mult != nullptr)
        SIREN_QUANT_TYPES(false, true);
    else
        SIREN_QUANT_TYPES(false, false);
#undef SIREN_QUANT_TYPES
#undef SIREN_QUANT
}

}  // namespace

void launch_fp8_quant(hipStream_t stream, const Fp8Quant& a) {
    if (!rows_only(a)) return launch_tiles(stream, a, nullptr);
    const int col_blocks = (int)fp8_blocks(a.cols);
    const int per = a.type == FP8_F32 ? ROWS_PER_GROUP<float> : ROWS_PER_GROUP<__bf16>;
    const int64_t groups = (a.rows + per - 1) / per * col_blocks;
#define SIREN_QUANT_ROWS(T, E)                                                                                           \
    hipLaunchKernelGGL((quant_rows_kernel<T, E>), dim3((unsigned)groups), dim3(256), 0, stream, (const T*)a.x, a.ld, a.rows, \
                       a.cols, a.q, a.s, col_blocks, a.panels)
    if (a.type == FP8_F32 && a.e5m2) SIREN_QUANT_ROWS(float, true);
    if (a.type == FP8_BF16 && a.e5m2) SIREN_QUANT_ROWS(__bf16, true);
    if (a.type == FP8_F16 && a.e5m2) SIREN_QUANT_ROWS(_Float16, true);
    if (a.type == FP8_F32 && !a.e5m2) SIREN_QUANT_ROWS(float, false);
    if (a.type == FP8_BF16 && !a.e5m2) SIREN_QUANT_ROWS(__bf16, false);
    if (a.type == FP8_F16 && !a.e5m2) SIREN_QUANT_ROWS(_Float16, false);
#undef SIREN_QUANT_ROWS
}

void launch_fp8_quant2(hipStream_t stream, const Fp8Quant& a, const Fp8Quant& b) {
    const bool alike = a.type == b.type && a.e5m2 == b.e5m2 && (a.mult != nullptr) == (b.mult != nullptr);
    if (alike && !rows_only(a) && !rows_only(b) && (int64_t)tiles_in(a) + tiles_in(b) <= 0xFFFFFF)
        return launch_tiles(stream, a, &b);
    launch_fp8_quant(stream, a);
    launch_fp8_quant(stream, b);
}

void launch_fp8_colsum(hipStream_t stream, const float* colsum, int64_t blocks, int64_t cols, float* out) {
    hipLaunchKernelGGL(colsum_kernel, dim3((unsigned)((cols + 31) / 32)), dim3(1024), 0, stream, colsum, blocks, cols, out);
}

}  // namespace siren
