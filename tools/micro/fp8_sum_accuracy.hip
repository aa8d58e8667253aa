// Micro-test: how exactly the matrix instructions sum products of e4m3 values: the scaled 16x16x128 fp8 form (scales of 1), the
// 16x16x32 fp8 form, and the 16x16x32 bf16 form on the same values, against sums in 64 bits. Products of two e4m3 values have 8
// bits of mantissa, so that 32-bit sums of exact products would be off by some 2^-24 of the summands' magnitudes each.
//   hipcc --offload-arch=gfx950 -O3 -Xclang -target-feature -Xclang -packed-fp32-ops tools/micro/fp8_sum_accuracy.hip -o <exe>
#include <hip/hip_runtime.h>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
enum { SCALED, PLAIN, BF16 };
const char* const NAME[3] = {"fp8 16x16x128 scaled", "fp8 16x16x32", "bf16 16x16x32"};

// d (16 x 16) = a b^T of a, b (16 x k): codes, or for the bf16 form their values. k is a multiple of 128; the order of k within
// an instruction is the same for both operands, which is all that a sum needs
template <int FORM>
__global__ void product(const uint8_t* a, const uint8_t* b, const float* fa, const float* fb, float* d, int k) {
    const int r = threadIdx.x & 15, g = threadIdx.x >> 4;
    f32x4 c = {};
    if constexpr (FORM == SCALED) {
        for (int at = 0; at < k; at += 128) {
            i32x8 x, y;
            for (int h = 0; h < 2; ++h) {
                const i32x4 p = *(const i32x4*)(a + r * k + at + 64 * h + 16 * g), q = *(const i32x4*)(b + r * k + at + 64 * h + 16 * g);
                for (int i = 0; i < 4; ++i) x[4 * h + i] = p[i], y[4 * h + i] = q[i];
            }
            c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 0, 0, 0, 127, 0, 127);
        }
    } else if constexpr (FORM == PLAIN) {
        for (int at = 0; at < k; at += 32)
            c = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(*(const long*)(a + r * k + at + 8 * g), *(const long*)(b + r * k + at + 8 * g), c,
                                                           0, 0, 0);
    } else {
        for (int at = 0; at < k; at += 32) {
            bf16x8 x, y;
            for (int i = 0; i < 8; ++i) x[i] = (__bf16)fa[r * k + at + 8 * g + i], y[i] = (__bf16)fb[r * k + at + 8 * g + i];
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
        }
    }
    for (int i = 0; i < 4; ++i) d[(4 * g + i) * 16 + r] = c[i];
}

#define OK(call) do { if ((call) != hipSuccess) { printf("failed: %s\n", #call); exit(1); } } while (0)

float value(int code) {
    const int m = code & 7, e = (code >> 3) & 15;
    return (code & 128 ? -1.f : 1.f) * (e ? ldexpf(1 + m / 8.f, e - 7) : ldexpf(m / 8.f, -6));
}
int nearest(float x) {  // of the finite codes
    int best = 0;
    for (int c = 0; c < 127; ++c)
        if (fabsf(value(c) - fabsf(x)) < fabsf(value(best) - fabsf(x))) best = c;
    return best | (x < 0 ? 128 : 0);
}

int main() {
    const int K = 8192, REPS = 8;
    uint8_t *a, *b;
    float *fa, *fb, *d;
    OK(hipMalloc(&a, 16 * K)); OK(hipMalloc(&b, 16 * K)); OK(hipMalloc(&fa, 64 * K)); OK(hipMalloc(&fb, 64 * K));
    OK(hipMalloc(&d, 1024));
    std::mt19937 gen(1);
    std::normal_distribution<float> normal;
    for (int whole = 0; whole < 2; ++whole)
        for (int k : {128, 1024, 8192}) {
            double err[3] = {}, all = 0, worst[3] = {};
            for (int rep = 0; rep < REPS; ++rep) {
                std::vector<uint8_t> ca(16 * k), cb(16 * k);
                std::vector<float> va(16 * k), vb(16 * k);
                for (int i = 0; i < 16 * k; ++i) {
                    ca[i] = nearest(whole ? (float)((int)(gen() % 17) - 8) : 60 * normal(gen));
                    cb[i] = nearest(whole ? (float)((int)(gen() % 17) - 8) : 60 * normal(gen));
                    va[i] = value(ca[i]), vb[i] = value(cb[i]);
                }
                OK(hipMemcpy(a, ca.data(), 16 * k, hipMemcpyHostToDevice)); OK(hipMemcpy(b, cb.data(), 16 * k, hipMemcpyHostToDevice));
                OK(hipMemcpy(fa, va.data(), 64 * k, hipMemcpyHostToDevice)); OK(hipMemcpy(fb, vb.data(), 64 * k, hipMemcpyHostToDevice));
                float got[3][256];
                product<SCALED><<<1, 64>>>(a, b, fa, fb, d, k);
                OK(hipMemcpy(got[0], d, 1024, hipMemcpyDeviceToHost));
                product<PLAIN><<<1, 64>>>(a, b, fa, fb, d, k);
                OK(hipMemcpy(got[1], d, 1024, hipMemcpyDeviceToHost));
                product<BF16><<<1, 64>>>(a, b, fa, fb, d, k);
                OK(hipMemcpy(got[2], d, 1024, hipMemcpyDeviceToHost));
                for (int i = 0; i < 256; ++i) {
                    double want = 0, mag = 0;
                    for (int c = 0; c < k; ++c) {
                        const double p = (double)va[i / 16 * k + c] * vb[i % 16 * k + c];
                        want += p, mag += fabs(p);
                    }
                    all += want * want;
                    for (int f = 0; f < 3; ++f) {
                        err[f] += (got[f][i] - want) * (got[f][i] - want);
                        worst[f] = fmax(worst[f], fabs(got[f][i] - want) / mag);
                    }
                }
            }
            for (int f = 0; f < 3; ++f)
                printf("%-8s k %5d  %-21s rms error %.1e of the rms result, worst %.1e of the summands' magnitudes\n",
                       whole ? "whole" : "normal", k, NAME[f], sqrt(err[f] / all), worst[f]);
        }
    return 0;
}
