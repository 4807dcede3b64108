// aih_kv.h -- the paged 8-bit KV cache (include/aihost_hip.h): argument checks
// on the host and what its kernels share.
#pragma once

#include "aih_internal.h"

namespace aih_kv {

constexpr int kMaxSeqs = 4096;   // requests per call: bounds the LDS tables of aih_kv_plan and the scans of the others

// The context's device for the length of a call; the caller's device again
// afterwards.
class DeviceGuard {
public:
    explicit DeviceGuard(int device)
    {
        status = hipGetDevice(&before);
        if (status == hipSuccess && before != device) {
            status = hipSetDevice(device);
            changed = status == hipSuccess;
        }
    }
    ~DeviceGuard()
    {
        if (changed) (void)hipSetDevice(before);
    }
    DeviceGuard(const DeviceGuard &) = delete;
    DeviceGuard &operator=(const DeviceGuard &) = delete;
    hipError_t status = hipSuccess;

private:
    int before = -1;
    bool changed = false;
};

constexpr int kMaxHeads = 65535;             // of keys and values, and of queries
constexpr int64_t kMaxGroups = 0xFFFFFF;     // workgroups of 256 threads of a launch: HIP counts threads in 32 bits

// The sizes of a cache description; the pointers are checked where they are used.
static inline int check_shape(const aih_kv_cache *kv)
{
    if (!kv || kv->reserved != 0 || kv->n_kv_heads <= 0 || kv->n_blocks <= 0) return AIH_E_INVALID;
    if (kv->format != AIH_KV_INT8 && kv->format != AIH_KV_E4M3) return AIH_E_UNSUPPORTED;
    if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256) return AIH_E_UNSUPPORTED;
    const int bt = kv->block_tokens;
    if (bt != 16 && bt != 32 && bt != 64 && bt != 128 && bt != 256) return AIH_E_UNSUPPORTED;
    const int64_t tokens = (int64_t)kv->n_blocks * bt;
    // slots are 32-bit, and so are the indices of 16-token groups and of a row's values
    if (tokens > 0x7FFFFFFF || kv->n_kv_heads > kMaxHeads || tokens / 16 * kv->n_kv_heads > 0x7FFFFFFF) return AIH_E_LIMIT;
    return AIH_OK;
}

static inline bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

static inline int check_cache(const aih_kv_cache *kv)
{
    const int rc = check_shape(kv);
    if (rc) return rc;
    if (!kv->k || !kv->v || !kv->k_scale || !kv->v_scale || !aligned16(kv->k) || !aligned16(kv->v)) return AIH_E_INVALID;
    if (reinterpret_cast<uintptr_t>(kv->k_scale) % 4 || reinterpret_cast<uintptr_t>(kv->v_scale) % 4)
        return AIH_E_INVALID;
    return AIH_OK;
}

static inline int log2_of(int v) { return 31 - __builtin_clz((unsigned)v); }

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

// Sum, inclusive scans and maximum over the 64 lanes on the DPP path (a shuffle
// goes through LDS, ten times the latency): within rows of 16, then row 0 into row 1
// and 2 into 3 (row_bcast:15), then rows 0, 1 into 2, 3 (row_bcast:31).  A lane
// that nothing is shifted into gets a zero.  `op` has to be associative, with 0 for its unit.
template <typename T, typename Op>
__device__ __forceinline__ T wave_scan(T v, Op op)
{
    const T zero = 0;
    v = op(v, __builtin_amdgcn_update_dpp(zero, v, 0x111, 0xF, 0xF, true));   // row_shr:1
    v = op(v, __builtin_amdgcn_update_dpp(zero, v, 0x112, 0xF, 0xF, true));
    v = op(v, __builtin_amdgcn_update_dpp(zero, v, 0x114, 0xF, 0xF, true));
    v = op(v, __builtin_amdgcn_update_dpp(zero, v, 0x118, 0xF, 0xF, true));
    v = op(v, __builtin_amdgcn_update_dpp(zero, v, 0x142, 0xA, 0xF, false));
    return op(v, __builtin_amdgcn_update_dpp(zero, v, 0x143, 0xC, 0xF, false));
}
__device__ __forceinline__ int32_t wave_scan(int32_t v)
{
    return wave_scan(v, [](int32_t a, int32_t b) { return a + b; });
}
__device__ __forceinline__ float wave_add(float v)
{
    v = wave_scan(v, [](float a, float b) { return a + b; });
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
    v = wave_scan(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

}  // namespace aih_kv
