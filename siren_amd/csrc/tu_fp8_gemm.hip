// tu_fp8_gemm.hip — the product of two 8-bit operands with block scales: out = act(A B^T + bias).
//
//   out[m][n] = sum_b sa[m][b] sb[n][b] sum_{k in block b} a[m][k] b[n][k], 32-bit sums
//
// The card's fp8 matrix instructions keep about 17 bits of the products that one instruction sums (rms errors of 1.5e-5 of
// the result on random operands, whatever the length; the bf16 ones 1e-8 to 1e-7: tools/micro/fp8_sum_accuracy.hip), the bf16
// ones lose nothing of these operands' products; an e4m3 value times a power of two is a bf16 number exactly, and
// v_cvt_scalef32_pk_bf16_fp8 makes two of them at once. So the operands travel as bytes through HBM and LDS, are scaled and
// widened in registers, and the bf16 matrix pipe sums them, for 16-bit results too (an output that nearly cancels would show the
// fp8 instructions' missing bits there as well).
// Exactly, that is, where bf16 reaches: of scale bytes 3 and more (e5m2: 10) every code is a bf16 number, its subnormal ones,
// which the pipe keeps, among them. Below, in blocks whose magnitudes stay under 2^-116 (e5m2: 2^-102), values under 2^-126 are
// rounded to multiples of 2^-133, the nearest, ties to even: off by 2^-134 at most. Above, a block whose largest magnitude
// rounds to 2^128 (from 2^128 (1 - 2^-5) on; e5m2: 2^-4) holds an infinity there, in fp32 as in bf16. A scale that is carried
// apart, into the 32-bit sums, would lose neither, for a multiplication of every sum in each block.
//
// A workgroup of 4 waves owns 256 x 128 of out (128 x 128 where rows are few), each wave 128 x 64 (64 x 64) in tiles of
// 32 x 32. Half a block, 64 k of both operands, is one stage of LDS: 24 KiB by direct global-to-LDS loads, three stages, so
// the loads run two half blocks ahead; two workgroups share a CU, and one's stores run behind the other's products (where there
// are more tiles than the 512 that the card holds at once: 512 begin, sum and store together). With 128
// rows two stages of 16 KiB, so that four workgroups share a CU (50001 x 832 x 320: 44 us with three stages, 42 with two).
// A half block of padding alone, and a wave whose rows or columns do not exist, take no products (42 -> 37 us).
//
// An LDS row is 64 bytes of one operand row; its 16-byte pieces are permuted by (row >> 2) & 3 on the way in, so that the 16
// lanes that read one piece of 16 rows hit distinct banks. The sums do not care in which order k is taken as long as both
// operands agree, so a lane's 16 contiguous bytes serve two instructions of 8.
#include <algorithm>
#include <cmath>

#include "fp8.h"
#include "fp8_device.h"
#include "siren_common.h"

namespace siren {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int TN = 128;  // columns of a workgroup's tile
constexpr int BK = 128;  // k of one block of scales
constexpr int HK = 64;   // k of one stage of LDS: half a block

struct GemmArgs {
    const uint8_t *a, *b, *sa, *sb;
    int64_t rsa, rsb, hsa, hsb;  // bytes from row to row, from half block to half block
    int64_t lsa, lsb;            // bytes of a row's scales
    int64_t m, n;
    int sha, shb;                // scales per row (0) or per 128 rows (7)
    int steps, steps_per_split;  // blocks of k, and of one split
    int halves;                  // half blocks with k in them
    int tiles_m, tiles_n;
    const float* bias;
    int act;
    float omega, turn, turn_low;  // turns = omega / 2 pi, in 32 bits and what they leave
    double turns;
    void* out;                   // split: fp32 partial products (splits, m, n)
    __bf16* deriv;
};

// Nontemporal: a result is read by a later kernel, after the operands that it would push out of L2 (262144 x 1024 x 1024
// fp32 out: 620 -> 550 us). Rows that begin anywhere but at 64 bytes leave lines that two stores share, which L2 has to join:
// 30000 x 1023 fp32 takes 58 us through L2, 96 nontemporal, 71 element by element; 14768 x 13240 bf16 174 and 338; with rows
// of 1008 fp32 (a multiple of 64 bytes, not of 128) it is 199 through L2 and 131.
// dst is global memory, which the compiler has to be told: a pointer out of a struct of arguments is generic to it, and a flat
// store counts as an access of LDS too, so that the epilogue's waits for LDS waited for memory
// (65536 x 256 x 256 bf16: 17.0 us, 13.8 with both this and the pacing of stores below).
template <typename T>
__device__ __forceinline__ void put4(T* dst, f32x4 v, int valid, bool once) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(1))) T Element;
    typedef __attribute__((address_space(1))) T4 Line;
    typedef __attribute__((address_space(1))) typename Quad<T>::Type Anywhere;
    const T4 h = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    if (once && valid >= 4) {
        __builtin_nontemporal_store(h, (Line*)dst);
    } else if (valid >= 4) {
        *(Anywhere*)dst = h;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < valid) ((Element*)dst)[k] = h[k];
    }
}

constexpr float MANY_TURNS = 4194304.f;  // 2^22: beyond, fp32 holds no whole number of turns and a fraction

// The phases omega z of four z, in turns, for v_sin_f32 and v_cos_f32: z (omega / 2 pi) less its whole turns, by fused steps
// with the factor in two parts, so that neither omega z nor the product is rounded on the way. Of phases past MANY_TURNS the
// fraction is taken in 64 bits: in a branch that the wave takes if any lane has one, where the others keep their result, so that
// no output depends on its neighbours. Chosen for each element, the 64-bit steps were issued whether a lane needed them or not
// (262144 x 1024 x 1024 with the sine 692 us, 670 then, both in the first passes after an idle card, which are slower than the
// later 590; 16384 x 1024 x 1024 bf16 40.2 with the phase first, 38.9).
__device__ __forceinline__ f32x4 turns4(const f32x4& z, const GemmArgs& g) {
    f32x4 u;
    float most = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float q = __builtin_rintf(z[k] * g.turn);
        u[k] = __builtin_fmaf(z[k], g.turn_low, __builtin_fmaf(z[k], g.turn, -q));
        most = fmaxf(most, __builtin_fabsf(q));
    }
    if (__builtin_expect(__any(most > MANY_TURNS), 0)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float w = (float)__builtin_amdgcn_fract((double)z[k] * g.turns);
            u[k] = __builtin_fabsf(__builtin_rintf(z[k] * g.turn)) > MANY_TURNS ? w : u[k];  // as above: by its own turns
        }
    }
    return u;
}

// bias, sine and the store of out[row][col .. col + 3], of which valid exist
template <typename T>
struct Finish {
    int64_t col;
    int valid;
    bool once, once16;  // rows of T, of 16 bits, begin at 64 bytes
    f32x4 bias;
    __device__ __forceinline__ Finish(const GemmArgs& g, int64_t c) : col(c) {
        valid = g.n - col < 4 ? (int)(g.n - col) : 4;
        once = (g.n * (int)sizeof(T) & 63) == 0;
        once16 = (g.n * 2 & 63) == 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) bias[k] = g.bias != nullptr && k < valid ? g.bias[col + k] : 0.f;
    }
    __device__ __forceinline__ void store(const GemmArgs& g, int64_t row, f32x4 v) const {
        v += bias;
        if (g.act == FP8_ACT_SINE) {
            const f32x4 u = turns4(v, g);
            if (g.deriv != nullptr) {
                f32x4 d;
#pragma unroll
                for (int k = 0; k < 4; ++k) d[k] = g.omega * __builtin_amdgcn_cosf(u[k]);
                put4(g.deriv + row * g.n + col, d, valid, once16);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = __builtin_amdgcn_sinf(u[k]);
        }
        put4((T*)g.out + row * g.n + col, v, valid, once);
    }
};

void set_omega(GemmArgs& g, float omega) {
    g.omega = omega;
    g.turns = (double)omega * 0.15915494309189533577;
    g.turn = (float)g.turns;
    g.turn_low = (float)(g.turns - (double)g.turn);
}

// The products of one half block (64 k) of a wave's RT x 2 tiles of 32 x 32, bytes to bf16 and scaled on the way, in four
// slices of 16 k: the next slice's widening (3 instructions a product at RT = 4) stands beside this one's products. (Placing
// them one by one with scheduling barriers was 2 % slower than the compiler's own order.)
template <bool E5M2A, int RT>
__device__ __forceinline__ void half_block(const uint8_t* la, const uint8_t* lb, int lane, const uint32_t (&ba)[RT],
                                           const uint32_t (&bb)[2], f32x16 (&acc)[RT][2]) {
    const int r = lane & 31, h = lane >> 5, sw = (r >> 2) & 3;
    // this lane's two 16-byte pieces of a row: piece 2 i + h of the row lies at (2 i + h) ^ sw
    const int at[2] = {r * HK + ((h ^ sw) * 16), r * HK + (((2 + h) ^ sw) * 16)};
    u32x4 ra[2][RT], rb[2][2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int j = 0; j < 2; ++j) rb[p][j] = *(const u32x4*)(lb + j * 32 * HK + at[p]);
#pragma unroll
        for (int i = 0; i < RT; ++i) ra[p][i] = *(const u32x4*)(la + i * 32 * HK + at[p]);
    }
    float fa[RT], fb[2];
#pragma unroll
    for (int i = 0; i < RT; ++i) fa[i] = __uint_as_float(ba[i] << 23);
#pragma unroll
    for (int j = 0; j < 2; ++j) fb[j] = __uint_as_float(bb[j] << 23);
    bf16x8 va[2][RT], vb[2][2];
    auto widen = [&](int k) {
        const int p = k >> 1, w = 2 * (k & 1), to = k & 1;
#pragma unroll
        for (int j = 0; j < 2; ++j) vb[to][j] = widen8<false>(rb[p][j][w], rb[p][j][w + 1], fb[j]);
#pragma unroll
        for (int i = 0; i < RT; ++i) va[to][i] = widen8<E5M2A>(ra[p][i][w], ra[p][i][w + 1], fa[i]);
    };
    widen(0);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (k < 3) widen(k + 1);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vb[k & 1][j], va[k & 1][i], acc[i][j], 0, 0, 0);
    }
}

template <typename T, bool E5M2A, bool SPLIT, int RT>
__global__ __launch_bounds__(256, 2) void gemm_kernel(GemmArgs g) {
    constexpr int TM = RT * 64;                 // rows of the workgroup's tile: 2 waves of RT x 32
    constexpr int STAGE = (TM + TN) * HK;       // bytes of one half block
    constexpr int LOADS = (TM + TN) / 16 / 4;   // 1 KiB pieces of it a wave loads
    constexpr int STAGES = RT == 2 ? 2 : 3;
    constexpr int ES = 68;                      // floats of an LDS row of the epilogue
    constexpr int PASS = RT / 2;                // tiles of 32 rows a wave stores at a time
    constexpr int STRIP = PASS * 32 * ES;       // floats of a wave's strip
    __shared__ __align__(16) uint8_t lds[STAGES * STAGE > STRIP * 16 ? STAGES * STAGE : STRIP * 16];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = wave & 1, wn = wave >> 1;

    // Workgroups go round-robin to the 8 dies: give each die a contiguous run of the (split, tile) list, columns fastest, so
    // that the tiles that share rows of A, or a split's k of both operands, meet in one L2 (the splits of a 1024 x 1024
    // product over 262144, dealt out tile by tile, read B from HBM on every die: 550 us instead of 455)
    const int tiles = g.tiles_m * g.tiles_n;
    int tile = blockIdx.x;
    {
        const int all = gridDim.x, per = all / 8, rest = all % 8, x = tile & 7, y = tile >> 3;
        tile = x * per + (x < rest ? x : rest) + y;
    }
    const int split = SPLIT ? __builtin_amdgcn_readfirstlane(tile / tiles) : 0;
    tile -= split * tiles;
    const int tm = __builtin_amdgcn_readfirstlane(tile / g.tiles_n), tn = tile - tm * g.tiles_n;
    const int64_t m0 = (int64_t)tm * TM, n0 = (int64_t)tn * TN;
    const int first = split * g.steps_per_split;
    const int last = first + g.steps_per_split < g.steps ? first + g.steps_per_split : g.steps;
    const int halves = (2 * last < g.halves ? 2 * last : g.halves) - 2 * first;
    const bool idle = m0 + wm * RT * 32 >= g.m || n0 + wn * 64 >= g.n;

    // This wave's 1 KiB pieces of a stage: 16 rows of A or of B each, lane / 4 the row, lane % 4 the place in LDS. Rows
    // past the operand's end read its last row; their products are not stored.
    const uint8_t* base[LOADS];
    int64_t step[LOADS];
    uint32_t off[LOADS];
    const int prow = lane >> 2, piece = (lane & 3) ^ ((prow >> 2) & 3);
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const int p = wave * LOADS + j;  // a piece is all A or all B: TM / 16 pieces of A
        const bool is_a = p < TM / 16;
        const int64_t row0 = is_a ? m0 : n0, rows = is_a ? g.m : g.n, rs = is_a ? g.rsa : g.rsb;
        const int64_t row = (is_a ? p * 16 : p * 16 - TM) + prow;
        step[j] = is_a ? g.hsa : g.hsb;
        base[j] = (is_a ? g.a : g.b) + row0 * rs + 2 * first * step[j];
        off[j] = (uint32_t)((row0 + row < rows ? row : rows - 1 - row0) * rs) + piece * 16;
    }
    const unsigned lds0 = lds_addr(lds);
    auto load = [&](int stage, int half) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
            glds_x4(base[j] + half * step[j], off[j], lds0 + stage * STAGE + (wave * LOADS + j) * 1024);
    };

    // the scales of this lane's rows, eight blocks of k in two words
    const uint8_t *qa[RT], *qb[2];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int64_t ra = m0 + (wm * RT + i) * 32 + (lane & 31);
        qa[i] = g.sa + ((ra < g.m ? ra : g.m - 1) >> g.sha) * g.lsa;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t rb = n0 + (wn * 2 + j) * 32 + (lane & 31);
        qb[j] = g.sb + ((rb < g.n ? rb : g.n - 1) >> g.shb) * g.lsb;
    }

    f32x16 acc[RT][2] = {};
    uint64_t wa[RT], wb[2];
    load(0, 0);
    if (STAGES == 3) load(1, 1);
    int stage = 0;
    for (int half = 0; half < halves; ++half) {
        const int block = first + (half >> 1);
        if (half == 0 || ((half & 1) == 0 && (block & 7) == 0)) {
            const int at = block & ~7, more = at + 4 < g.lsa ? at + 4 : at;
#pragma unroll
            for (int i = 0; i < RT; ++i)
                wa[i] = *(const uint32_t*)(qa[i] + at) | (uint64_t) * (const uint32_t*)(qa[i] + more) << 32;
#pragma unroll
            for (int j = 0; j < 2; ++j)
                wb[j] = *(const uint32_t*)(qb[j] + at) | (uint64_t) * (const uint32_t*)(qb[j] + more) << 32;
            // vmcnt(0), here and not at their first use: hipcc does not count the direct-to-LDS loads, so its own wait in
            // the loop's body would be for all of those, every half block
            __builtin_amdgcn_s_waitcnt(0x0F70);
        }
        // This stage's loads are in. With three stages the next one's, issued later, may be under way: loads return in order,
        // and at the last stage there are no newer ones. This wave's own reads of the stage before are done too.
        if (STAGES == 3 && half + 1 < halves)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        // every wave's are in, and every wave has read the stage before this one, which the next loads overwrite
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (half + STAGES - 1 < halves) load(stage == 0 ? STAGES - 1 : stage - 1, half + STAGES - 1);
        const int shift = 8 * (block & 7);
        uint32_t ba[RT], bb[2];
#pragma unroll
        for (int i = 0; i < RT; ++i) ba[i] = (uint32_t)(wa[i] >> shift) & 0xFFu;
#pragma unroll
        for (int j = 0; j < 2; ++j) bb[j] = (uint32_t)(wb[j] >> shift) & 0xFFu;
        const uint8_t* la = lds + stage * STAGE + wm * RT * 32 * HK;
        const uint8_t* lb = lds + stage * STAGE + (TM + wn * 64) * HK;
        if (!idle) half_block<E5M2A, RT>(la, lb, lane, ba, bb, acc);
        stage = stage == STAGES - 1 ? 0 : stage + 1;
    }

    // B rows are the instruction's rows: registers 4 k .. 4 k + 3 of a 32 x 32 tile are out[lane % 32][8 k + 4 (lane / 32) ..].
    // They pass through LDS (the wave's quarter of the stages, which no one reads any more), half of the wave's rows at a time,
    // so that 16 lanes store the wave's 64 columns of one row: stored as they lie, 32 bytes a row, they cost HBM twice the
    // requests, and with 32 columns at a time rows of odd widths left twice the shared lines (174691 x 344 x 1282 fp32: 411 us,
    // now 319). The loop over the rows also keeps the epilogue short; unrolled over the accumulators it outgrew the
    // instruction cache.
    float* strip = (float*)lds + wave * STRIP;
    __syncthreads();
    const int64_t wave_m = m0 + wm * RT * 32;
    const int sub = lane >> 4, quad = (lane & 15) * 4;
    const int64_t col = n0 + wn * 64 + quad;
    const Finish<T> to(g, col);
#pragma unroll
    for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int i = 0; i < PASS; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const f32x16& from = acc[p * PASS + i][j];
                    *(f32x4*)(strip + (i * 32 + (lane & 31)) * ES + j * 32 + 8 * k + 4 * (lane >> 5)) =
                        f32x4{from[4 * k], from[4 * k + 1], from[4 * k + 2], from[4 * k + 3]};
                }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (col < g.n) {
            for (int row = sub; row < PASS * 32; row += 16) {  // four rows' reads before the first is stored
                // Eight of a wave's stores under way and no more: a burst of all 32 stands before the loads of the workgroup
                // that shares the CU (262144 x 1024 x 1024 fp32 526 us, paced 510; 50001 x 832 x 320 bf16 37.5 and 35.4)
                asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
                f32x4 v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = *(const f32x4*)(strip + (row + 4 * u) * ES + quad);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int64_t m = wave_m + p * PASS * 32 + row + 4 * u;
                    if (m < g.m) {
                        if constexpr (SPLIT)
                            put4((float*)g.out + (split * g.m + m) * g.n + col, v[u], to.valid, to.once);
                        else
                            to.store(g, m, v[u]);
                    }
                }
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// A layer of a few rows (up to 32) in one launch: what it cannot do without is the weight's bytes. A wave owns NT x 16
// columns, a workgroup four times as many: it asks for its weights of FEW_K k first, all waves round that much of x to 8
// bits into LDS while they travel (half a wave a block), then the wave's rows of the weight times the rows of x, 16 at a
// time. Rows of x that do not exist are whatever LDS holds: an output depends on its own row only. 65536 columns of 256:
// 6 us for one row (16.8 MB: 2.8 TB/s), 9 for 32 (8.4 MB of results more).
constexpr int FEW_ROWS = 32, FEW_K = 512;
struct FewArgs {
    const void* x;
    int64_t ld, m, k;
    const uint8_t *w, *sw;
    GemmArgs out;  // n, bias, act, omega, out
};
//
// KW = 4: the waves share 16 columns and split k, 2048 of it at a time, and add their sums in order through LDS: a quarter
// of the steps where the columns alone do not fill the card (1 row, 4096 -> 1024: 16.8 us, 8.8).
template <typename T, int MT, int NT, int KW>
__global__ __launch_bounds__(256) void few_rows_kernel(FewArgs f) {
    constexpr int CHUNK = FEW_K / 128, ALL = CHUNK * KW;  // blocks of a wave, of the workgroup
    constexpr int LD = ALL * 128 + 16;                    // LDS rows 16 bytes apart from a bank period
    __shared__ __align__(16) uint8_t xq[MT * 16 * LD];
    __shared__ uint8_t xs[MT * 16 * ALL];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 15, q = lane >> 4;
    const GemmArgs& g = f.out;
    const int64_t n0 = (KW == 1 ? (int64_t)blockIdx.x * 4 + wave : (int64_t)blockIdx.x) * (NT * 16);
    const int own = KW == 1 ? 0 : wave * CHUNK;  // the wave's first block among the workgroup's
    const int64_t kp = (f.k + 127) / 128 * 128;
    const int blocks = (int)(kp / 128);
    const uint8_t *w[NT], *sw[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {  // columns past the end read the last one's weights and store nothing
        const int64_t row = n0 + j * 16 + r < g.n ? n0 + j * 16 + r : g.n - 1;
        w[j] = f.w + row * kp + q * 16;
        sw[j] = f.sw + (row >> 7) * ((blocks + 3) / 4 * 4);
    }
    f32x4 acc[MT][NT] = {};
    for (int b0 = 0; b0 < blocks; b0 += ALL) {
        const int here = blocks - b0 < ALL ? blocks - b0 : ALL;             // blocks of the workgroup
        const int mine = here - own < CHUNK ? here - own : CHUNK;           // of the wave; none or fewer: nothing
        u32x4 wv[NT][CHUNK][2];
        uint32_t scales[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            scales[j] = mine > 0 ? *(const uint32_t*)(sw[j] + b0 + own) : 0u;
#pragma unroll
            for (int b = 0; b < CHUNK; ++b)
                if (b < mine) {
                    wv[j][b][0] = *(const u32x4*)(w[j] + (b0 + own + b) * 128);
                    wv[j][b][1] = *(const u32x4*)(w[j] + (b0 + own + b) * 128 + 64);
                }
        }
        if (b0 > 0) __syncthreads();  // x of the chunk before has been read
        // units of one block of one row, BATCH of a half wave's loaded before the first is rounded
        constexpr int BATCH = MT == 1 && KW == 1 ? 2 : 8;
        const int c4 = threadIdx.x & 31, half = threadIdx.x >> 5, all = (int)f.m * here;
        for (int u0 = half; u0 < all; u0 += 8 * BATCH) {
            float v[BATCH][4];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int u = u0 + 8 * i, row = u / here, b = u - row * here;
                const int64_t c0 = (int64_t)(b0 + b) * 128 + c4 * 4, left = f.k - c0;
                load_quad((const T*)f.x + row * f.ld + c0, u < all && left > 0 ? (left < 4 ? (int)left : 4) : 0, v[i]);
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int u = u0 + 8 * i, row = u / here, b = u - row * here;
                const int byte = exponent_byte<false>(half_wave_amax(v[i][0], v[i][1], v[i][2], v[i][3]));
                if (u < all) {
                    *(uint32_t*)(xq + row * LD + b * 128 + c4 * 4) =
                        pack4<false>(v[i][0], v[i][1], v[i][2], v[i][3], scale_of(byte));
                    if (c4 == 0) xs[row * ALL + b] = (uint8_t)byte;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int b = 0; b < CHUNK; ++b) {
            if (b < mine) {
                bf16x8 xf[MT][4];
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const int row = t * 16 + r;
                    const float fx = scale_of(xs[row * ALL + own + b]);
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        const u32x4 c = *(const u32x4*)(xq + row * LD + (own + b) * 128 + p * 64 + q * 16);
                        xf[t][2 * p] = widen8<false>(c[0], c[1], fx);
                        xf[t][2 * p + 1] = widen8<false>(c[2], c[3], fx);
                    }
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const float fw = scale_of((scales[j] >> (8 * b)) & 0xFFu);
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        const u32x4& c = wv[j][b][p >> 1];
                        const bf16x8 wf = widen8<false>(c[2 * (p & 1)], c[2 * (p & 1) + 1], fw);
#pragma unroll
                        for (int t = 0; t < MT; ++t)
                            acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, xf[t][p], acc[t][j], 0, 0, 0);
                    }
                }
            }
        }
    }
    if constexpr (KW > 1) {
        static_assert(NT == 1 && MT * 16 * LD >= KW * MT * 1024, "a wave's sums fit its share of x");
        __syncthreads();  // x has been read
        f32x4* red = (f32x4*)xq;
#pragma unroll
        for (int t = 0; t < MT; ++t) red[(wave * MT + t) * 64 + lane] = acc[t][0];
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int k = 1; k < KW; ++k) acc[t][0] += red[(k * MT + t) * 64 + lane];
    }
    // the weight's rows are the instruction's rows: lane (r, q) holds y[r][n0 + 16 j + 4 q ..]
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int64_t col = n0 + j * 16 + 4 * q;
        if (col < g.n) {
            const Finish<T> to(g, col);
#pragma unroll
            for (int t = 0; t < MT; ++t)
                if (t * 16 + r < f.m) to.store(g, t * 16 + r, acc[t][j]);
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
            if (col + 4 <= g.n) {
#pragma unroll 8
                for (int s = lo; s < hi; ++s) v += *(const Quad<float>::Type*)(src + s * plane);
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
        if (grp == 0 && i < total) Finish<T>(g, col).store(g, row, v);
    }
}

template <typename T>
void launch_join(hipStream_t stream, const GemmArgs& g, const void* part, int splits) {
    const int64_t quads = g.m * ((g.n + 3) / 4);
    // 8 waves a CU of one thread a quad are 131072 quads; below that, threads share them
    const int groups = quads >= 131072 || splits < 4 ? 1 : quads >= 16384 || splits < 16 ? 4 : 16;
    const int64_t want = (quads + 256 / groups - 1) / (256 / groups);
    const dim3 grid((unsigned)(want < 8192 ? want : 8192));
    if (groups == 16)
        hipLaunchKernelGGL((join_kernel<T, 16>), grid, dim3(256), 0, stream, g, (const float*)part, splits);
    else if (groups == 4)
        hipLaunchKernelGGL((join_kernel<T, 4>), grid, dim3(256), 0, stream, g, (const float*)part, splits);
    else
        hipLaunchKernelGGL((join_kernel<T, 1>), grid, dim3(256), 0, stream, g, (const float*)part, splits);
}

// Tiles of 256 rows need a third less of the operands' bytes; those of 128 leave less of a tile outside the result, and four
// workgroups of them share a CU, which hides a short sum's beginning and end.
int64_t tiles_of(int64_t m, int64_t n, int rows) { return (m + rows - 1) / rows * ((n + TN - 1) / TN); }
bool less_waste(int64_t m) { return 10 * ((m + 255) / 256 * 256) > 11 * ((m + 127) / 128 * 128); }  // by 128 rows, over 10 %

// 262144 x 1024 x 1024: 590 us with 256 rows, 607 with 128; 16384 x 4096 x 4096: 453 and 491; 50001 x 832 x 320: 48 and 37.
// At the borders, whole layers of bf16 rows with their rounding: 16384 x 1024 x 1024 (512 tiles) 46.3 and 48.0 us, 12288 rows of
// it (384 tiles) 41.1 and 38.2; k = 768 37.7 and 38.4, of 65536 rows 134 and 134, with the sine 41.3 and 41.1, 146 and 142; k =
// 512 of 65536 rows 99 and 97, with the sine 111 and 106
bool tall(int64_t m, int64_t n, int64_t k) { return k >= 1024 && tiles_of(m, n, 256) >= 512 && !less_waste(m); }

// A product whose tiles do not fill the card splits its k axis, where that pays for the partial results' way through memory
// and a second launch. By what was measured, in us: a block of k takes a workgroup of 128 rows 1.1, and 0.84 for each of those
// that share its CU; the join 5, and each split's m n floats 1.6e-6 m n written and read. Two workgroups a CU at most (more
// gained nothing). Split and whole: 200 x 200 x 1024 11 and 13, x 2048 12 and 22; 33 x 200 x 700 10.7 and 9.7, 2000 x 1000 x
// 1024 24 and 14, x 2048 33 and 22. 1000 x 1000 x 4000 in 4, 16 and 1: 25, 32 and 29 us.
struct Plan {
    int splits;
    bool tall;  // 256 rows a tile: sums of 64 blocks a workgroup and more (1024 x 1024 x 262144: 458 us and 525)
};
Plan plan_of(int64_t m, int64_t n, int64_t k) {
    const int64_t tiles = tiles_of(m, n, 128), tall_tiles = tiles_of(m, n, 256), steps = fp8_blocks(k);
    if (tiles >= 256 || steps < 4) return {1, tall(m, n, k)};
    int64_t splits = 1;
    bool rows256 = false;
    if (m > 128 && !less_waste(m) && steps * tall_tiles >= 64 * 512) {
        splits = 512 / tall_tiles;
        rows256 = true;
    } else {
        const double plane = 1.6e-6 * (double)m * (double)n;
        auto cost = [&](int64_t s) {
            const double shared = 0.84 * (double)((tiles * s + 255) / 256);
            return (double)((steps + s - 1) / s) * (shared > 1.1 ? shared : 1.1) + (s > 1 ? 5.0 + (double)s * plane : 0.0);
        };
        // the best number if a CU never had two, the largest that keeps it so, and 1
        int64_t best = (int64_t)std::sqrt(1.1 * (double)steps / plane);
        for (int64_t s : {std::min(best, 512 / tiles), std::min(best, 256 / tiles)}) {
            s = std::min(s, steps / 2);
            if (s > 1 && cost(s) < cost(splits)) splits = s;
        }
    }
    const int64_t per = (steps + splits - 1) / splits;
    return {(int)((steps + per - 1) / per), rows256};
}

template <typename T, bool E5M2A, bool SPLIT>
void launch_gemm(hipStream_t stream, GemmArgs& g, int splits, bool rows256) {
    g.tiles_m = (int)((g.m + (rows256 ? 255 : 127)) / (rows256 ? 256 : 128));
    g.tiles_n = (int)((g.n + TN - 1) / TN);
    const dim3 grid((unsigned)(g.tiles_m * g.tiles_n * splits));
    if (rows256)
        hipLaunchKernelGGL((gemm_kernel<T, E5M2A, SPLIT, 4>), grid, dim3(256), 0, stream, g);
    else
        hipLaunchKernelGGL((gemm_kernel<T, E5M2A, SPLIT, 2>), grid, dim3(256), 0, stream, g);
}

}  // namespace

// One launch, or rounding, product and join. Each workgroup of the one rounds all of x, four rows of 2048 k in a round trip of
// 3.3 us; the three take 14 us whatever the size. Columns 1024, one launch and three: 1 row of 4096 8.8 and 14.8 us, of 16384
// 29 and 15.6; 9 rows of 2048 9.9 and 15.0, of 4096 17.4 and 14.8; 16 rows of 2048 11.7 and 14.6; 32 rows of 512 7.9 and 11.9,
// of 1024 13.6 and 14.5, of 2048 25.7 and 14.9, 30 rows of 999 in bf16 21 and 15. Where the columns fill the card it reads the
// weight's bytes as fast: 30000 x 16384 with 4 rows 110 and 130 us.
bool fp8_few_rows(int64_t m, int64_t n, int64_t k) {
    const bool wide = n >= 64 * 256;
    if (m > 16) return m <= FEW_ROWS && k <= FEW_K;
    return (m + 3) / 4 * ((k + 2047) / 2048) <= 4 || (wide && m <= 4);
}

void launch_fp8_few_rows(hipStream_t stream, const void* x, int type, int64_t ld, int64_t m, int64_t k, const uint8_t* w,
                         const uint8_t* sw, int64_t n, const float* bias, int act, float omega, void* y, void* deriv) {
    FewArgs f = {};
    f.x = x;
    f.ld = ld;
    f.m = m;
    f.k = k;
    f.w = w;
    f.sw = sw;
    f.out.m = m;
    f.out.n = n;
    f.out.bias = bias;
    f.out.act = act;
    set_omega(f.out, omega);
    f.out.out = y;
    f.out.deriv = (__bf16*)deriv;
    // 32 columns a wave where that still is a workgroup a CU: half the rounding of x. A long k whose columns fill fewer CUs is
    // split among a workgroup's waves
    const bool two = n >= 128 * 256, split = m <= 16 && k > FEW_K && n < 64 * 256;
    const int columns = split ? 16 : two ? 128 : 64;
    const dim3 grid((unsigned)((n + columns - 1) / columns));
#define SIREN_FEW(T)                                                                                \
    do {                                                                                            \
        if (split)                                                                                  \
            hipLaunchKernelGGL((few_rows_kernel<T, 1, 1, 4>), grid, dim3(256), 0, stream, f);       \
        else if (m <= 16 && two)                                                                    \
            hipLaunchKernelGGL((few_rows_kernel<T, 1, 2, 1>), grid, dim3(256), 0, stream, f);       \
        else if (m <= 16)                                                                           \
            hipLaunchKernelGGL((few_rows_kernel<T, 1, 1, 1>), grid, dim3(256), 0, stream, f);       \
        else if (two)                                                                               \
            hipLaunchKernelGGL((few_rows_kernel<T, 2, 2, 1>), grid, dim3(256), 0, stream, f);       \
        else                                                                                        \
            hipLaunchKernelGGL((few_rows_kernel<T, 2, 1, 1>), grid, dim3(256), 0, stream, f);       \
    } while (0)
    if (type == FP8_F32) SIREN_FEW(float);
    if (type == FP8_BF16) SIREN_FEW(__bf16);
    if (type == FP8_F16) SIREN_FEW(_Float16);
#undef SIREN_FEW
}

int64_t fp8_product_ws_bytes(int64_t m, int64_t n, int64_t k) {
    const int s = plan_of(m, n, k).splits;
    return s > 1 ? (int64_t)s * m * n * 4 : 0;
}

void launch_fp8_product(hipStream_t stream, const Fp8Product& p) {
    GemmArgs g;
    g.a = p.a.data;
    g.b = p.b.data;
    g.sa = p.a.scale;
    g.sb = p.b.scale;
    g.rsa = p.a.panels ? HK : fp8_padded(p.k);
    g.rsb = p.b.panels ? HK : fp8_padded(p.k);
    g.hsa = p.a.panels ? p.a.rows * HK : HK;
    g.hsb = p.b.panels ? p.b.rows * HK : HK;
    g.lsa = g.lsb = fp8_scale_cols(p.k);
    g.m = p.a.rows;
    g.n = p.b.rows;
    g.sha = p.a.shift;
    g.shb = p.b.shift;
    g.steps = (int)fp8_blocks(p.k);
    g.halves = (int)((p.k + HK - 1) / HK);
    g.bias = p.bias;
    g.act = p.act;
    set_omega(g, p.omega);
    g.deriv = (__bf16*)p.deriv;
    const Plan plan = plan_of(g.m, g.n, p.k);
    const int splits = plan.splits;
    g.steps_per_split = (g.steps + splits - 1) / splits;
    g.out = splits > 1 ? p.ws : p.out;
    if (splits > 1) {
        if (p.e5m2_a)
            launch_gemm<float, true, true>(stream, g, splits, plan.tall);
        else
            launch_gemm<float, false, true>(stream, g, splits, plan.tall);
        g.out = p.out;
        if (p.type == FP8_F32) launch_join<float>(stream, g, p.ws, splits);
        if (p.type == FP8_BF16) launch_join<__bf16>(stream, g, p.ws, splits);
        if (p.type == FP8_F16) launch_join<_Float16>(stream, g, p.ws, splits);
        return;
    }
    if (p.e5m2_a) {
        if (p.type == FP8_F32) launch_gemm<float, true, false>(stream, g, 1, plan.tall);
        if (p.type == FP8_BF16) launch_gemm<__bf16, true, false>(stream, g, 1, plan.tall);
        if (p.type == FP8_F16) launch_gemm<_Float16, true, false>(stream, g, 1, plan.tall);
    } else {
        if (p.type == FP8_F32) launch_gemm<float, false, false>(stream, g, 1, plan.tall);
        if (p.type == FP8_BF16) launch_gemm<__bf16, false, false>(stream, g, 1, plan.tall);
        if (p.type == FP8_F16) launch_gemm<_Float16, false, false>(stream, g, 1, plan.tall);
    }
}

}  // namespace siren
