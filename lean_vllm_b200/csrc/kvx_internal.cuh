// What the library's sources share: error reporting, launch accounting, per-device facts, the store's destination
// table, and the small device functions around mbarriers and programmatic launches.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include <nvtx3/nvToolsExt.h>

#include "kvx.h"

namespace kvx {

// ------------------------------------------------------------------------------------------------ host side

// Records the calling thread's last error (kvx_last_error) and returns `code`.
int fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));

#define KVX_CUDA(call)                                                                                            \
    do {                                                                                                          \
        cudaError_t e_ = (call);                                                                                  \
        if (e_ != cudaSuccess) return kvx::fail(KVX_ERR_CUDA, "%s failed: %s", #call, cudaGetErrorString(e_));    \
    } while (0)

void count_launch();  // one kernel more for kvx_launch_count

// An NVTX range around each entry point that launches work, so a timeline (nsys, ncu's range view) shows which call
// queued which kernels. Without a tool attached, NVTX calls are no-ops.
struct Range {
    explicit Range(const char *name) { nvtxRangePushA(name); }
    ~Range() { nvtxRangePop(); }
};

struct Device {
    int index;
    int sms;
    int32_t *error_word;  // the device's diagnostic word (kvx_device_error)
};
int current_device(Device *out);

// ------------------------------------------------------------------------------------------------ status

// Errors kernels record, as bits: a copy's bounded wait ran out (its bytes did not all land), a store slot or
// block id past its cache (skipped), the wait self-test gave up, a position past its rotary table, a bounded wait of
// an attention launch ran out. Each goes into the launch's status word, when it has one, and into the device's
// diagnostic word (read and cleared by kvx_device_error).
constexpr int kErrCopyWait = 1;
constexpr int kErrPastCache = 2;
constexpr int kErrSelftest = 4;
constexpr int kErrPosition = 8;
constexpr int kErrAttentionWait = 16;

// Records `code` for a launch. The status word is mapped host memory, which no atomic reaches: it gets a plain store,
// so a launch that meets faults of two kinds reports the later one there, and both in the device's word.
__device__ __forceinline__ void flag_error(int32_t *error_word, int32_t *status, int code) {
    atomicOr(error_word, code);
    if (status) *reinterpret_cast<volatile int32_t *>(status) = code;
}

// ------------------------------------------------------------------------------------------------ store destinations

constexpr int kMaxStoreDests = 9;  // the local cache and up to 8 decode ranks

struct StoreDest {
    uint64_t k, v;
    int64_t block_stride, token_stride, head_stride;
    const void *slots;
    const int32_t *block_map;
    int32_t block_size, num_blocks, slot_bytes, src_first_head, num_heads, dst_first_head, block_map_len;
    int32_t block_shift;  // log2(block_size) when it is a power of two (the usual 16, 64, 256), else -1
};

// Checks `n_dests` destinations of rows with `num_heads` heads and lays them out for a kernel. ORs the addresses and
// strides that bound the alignment of what is written into `align_bits`.
int fill_dests(const kvx_store_dest *dests, int n_dests, int num_tokens, int num_heads, bool has_value, StoreDest *out,
               uint64_t *align_bits);

// ------------------------------------------------------------------------------------------------ device side

__device__ __forceinline__ uint64_t globaltimer() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

__device__ __forceinline__ uint32_t smem_u32(const void *p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}

// Two 32-bit operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// Programmatic stream serialization: lets the next such launch on the stream start, and waits until the kernels
// before this one have completed and their memory is visible.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_prerequisites() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

}  // namespace kvx
