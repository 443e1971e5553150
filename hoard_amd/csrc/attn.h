// Internal launch interface between the C ABI of a layer's attention half (attn.cpp)
// and its kernels.  Arguments are checked by attn.cpp.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "hoard_attn.h"

namespace hoard {

hipError_t launch_heads(const hoard_heads_args &a, hipStream_t s);
// Groups of tokens whose partial sums of dw_q and dw_k the workspace holds.
int heads_groups(const hoard_heads_args &a);
hipError_t launch_heads_grad(const hoard_heads_args &a, const hoard_heads_grads &g, float *work, hipStream_t s);

struct KvReadArgs {
    hoard_kv_cache c;
    int type, n_tokens;
    const int32_t *slots;
    void *k, *v;  // or NULL
    int64_t k_stride, v_stride;
};
hipError_t launch_kv_read(const KvReadArgs &a, hipStream_t s);

size_t attn_work_bytes(const hoard_kv_cache &c, const hoard_attn_args &a);
hipError_t launch_attn(const hoard_kv_cache &c, const hoard_attn_args &a, float *work, hipStream_t s);

}  // namespace hoard
