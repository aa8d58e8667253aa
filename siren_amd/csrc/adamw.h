// adamw.h — the host side of the many-tensor AdamW step (tu_adamw.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace siren {

constexpr int ADAMW_TENSORS = 104;      // tensors a launch: 36 bytes each of the 4 KiB of kernel arguments
constexpr int ADAMW_NORM_BLOCKS = 512;  // workgroups (and partial sums) of one norm launch: 2 a CU
constexpr int ADAMW_BLOCKS = 4096;      // workgroups of one update launch

struct AdamwHyper {
    double lr, b1, b2, max_norm;
    float omb1, b2f, omb2, epsf, decay;  // 1 - b1, b2, 1 - b2, eps, 1 - lr wd, rounded once
    uint64_t seed;
};

struct AdamwCall {
    int64_t count;
    void* const* p;
    const void* const* g;
    const int64_t* numel;
    const int32_t* dtype;  // 0 fp32, 1 bf16, 2 fp16
    int bits;              // 32 or 8
    void *m, *v;
    uint8_t *sm, *sv;
    int64_t* step;
    int64_t* counts;  // nullable: each tensor's own number of steps
    AdamwHyper h;
    void* scratch;
};

int64_t adamw_scratch_bytes(int64_t count);
void launch_adamw(hipStream_t st, const AdamwCall& call);

}  // namespace siren
