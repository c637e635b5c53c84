// What the attention kernels share: a launch's parameters, the mask, and the joining of partial results.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "kvx_internal.cuh"

namespace kvx {

constexpr float kLog2e = 1.4426950408889634f;

struct AttnParams {
    uint64_t query, out, k_cache, v_cache;
    int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;  // bytes
    int64_t block_stride, token_stride, head_stride;                           // bytes
    const int32_t *block_tables, *kv_lens, *q_starts, *prefix_lens;
    const float *slopes;
    int64_t table_stride;
    int32_t block_size, block_shift, num_blocks, max_blocks;  // block_shift: log2 of a power-of-two size, else -1
    int32_t batch, num_tokens, q_heads, kv_heads, group;      // group: query heads a KV head
    int32_t token0;  // of the call's tokens, the launch's first: queries, output and partial results begin there
    int32_t window;
    float scale, softcap;
    // Tokens that every sequence has in front of its own (rows see all of them), in blocks of their own; none when
    // their part arrives as partial results.
    const int32_t *shared_table;
    int32_t shared_len;
    int32_t *counters;
    float *partial_o;    // [slot][row of the tile][dim]
    float2 *partial_ml;  // [slot][row of the tile]: running maximum (log2 domain) and sum
    // Partial results of attention_tiles, [split][query token][head]: for rows whose keys it split, and for a shared
    // prefix, behind whose prefix_splits parts attention_rows leaves its own when there are any.
    float *split_o;
    float2 *split_ml;
    int32_t prefix_splits;
    // attention_rows takes the sequences of up to rows_limit query rows (query tokens x group), attention_tiles the rest.
    int32_t rows_limit;
    int32_t *status, *error_word;
};

// Which devices a kernel has its dynamic shared memory allowed on: asked for once per device, not per launch.
struct AllowedSmem {
    std::atomic<bool> on[64] = {};
    template <class Kernel>
    int allow(Kernel kernel, int bytes, int device) {
        if (device < 64 && on[device].load(std::memory_order_relaxed)) return KVX_OK;
        KVX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        if (device < 64) on[device].store(true, std::memory_order_relaxed);
        return KVX_OK;
    }
};

// Where a call's kernels are launched; serial: each after the one before it, with no overlap.
struct Queue {
    cudaStream_t stream;
    bool serial;
};

template <class Kernel, class... Args>
int launch(Kernel kernel, int64_t grid, int threads, int smem, const Queue &queue, const Args &...args) {
    if (grid > 0x7fffffff) return fail(KVX_ERR_INVALID, "more rows than a launch holds");
    cudaLaunchConfig_t cfg = {};
    cfg.stream = queue.stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = queue.serial ? 0 : 1;
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    KVX_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    count_launch();
    return KVX_OK;
}

// attention_tiles (attention_tiles.cu). `prefix_only`: all query rows against the shared prefix alone; else each
// sequence's rows above rows_limit. `groups`: tiles of rows per CTA, 1 or 2. It leaves `splits` parts to join, and finished
// rows when there is one split and it is not prefix_only.
int launch_tiles(const AttnParams &p, int head_dim, int dtype, bool mods, bool prefix_only, int groups, int splits,
                 const Device &device, const Queue &queue);
// The tokens of this cache that one of attention_tiles' copies brings; 0 if it cannot take the call (blocks that are no
// multiple of 8 tokens, strides that no tensor map holds, groups beyond a tile's rows).
int tile_box(const AttnParams &p);

constexpr int kMaxRowCtas = 1024;       // of attention_rows: a counter and two slots of partial results each
constexpr int kTileCounter = 8192;      // attention_tiles' counter, on a line of its own
constexpr int kRowTile = 16;            // rows of attention_rows' widest tile
constexpr int kTileKeys = 128;
constexpr int64_t kSplitRows = 131072;  // rows of partial results the workspace holds

// A sequence's query rows among the launch's and cached tokens (a shared prefix's first), with its lengths brought into
// range. Of one whose last query tokens are another launch's, the keys end with those that are here.
struct Sequence {
    int32_t q0, q_len, kv_len, prefix;
};

__device__ __forceinline__ Sequence sequence_of(const AttnParams &p, int s) {
    Sequence q;
    const int32_t begin = (p.q_starts ? p.q_starts[s] : s) - p.token0;
    const int32_t end = p.q_starts ? p.q_starts[s + 1] - p.token0 : begin + 1;
    q.q0 = max(begin, 0);
    q.q_len = max(0, min(end, p.num_tokens) - q.q0);
    const int64_t room = (int64_t)p.max_blocks * p.block_size;
    q.kv_len = (int32_t)min((int64_t)max(p.kv_lens[s], 0), room) + p.shared_len - max(0, end - p.num_tokens);
    q.prefix = p.prefix_lens ? min(max(p.prefix_lens[s], 0), q.kv_len) : p.shared_len;
    return q;
}

// Whose query token `token` is: the last sequence that starts at or before it.
__device__ __forceinline__ int sequence_at(const AttnParams &p, int token) {
    token += p.token0;
    if (!p.q_starts) return token;
    int low = 0, high = p.batch;
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (p.q_starts[mid] <= token) low = mid;
        else high = mid;
    }
    return low;
}

// Where sequence s keeps token t: a byte offset from the caches' first block and head, or -1 for a block id outside
// the cache, which is flagged.
__device__ __forceinline__ int64_t token_at(const AttnParams &p, int s, int32_t t) {
    const int32_t *table = p.block_tables + (int64_t)s * p.table_stride;
    if (t < p.shared_len) {
        table = p.shared_table;
    } else {
        t -= p.shared_len;
    }
    const int32_t b = p.block_shift >= 0 ? t >> p.block_shift : t / p.block_size;
    const int32_t id = table[b];
    if (id < 0 || id >= p.num_blocks) {
        flag_error(p.error_word, p.status, kErrPastCache);
        return -1;
    }
    return (int64_t)id * p.block_stride + (int64_t)(t - b * p.block_size) * p.token_stride;
}

// The first key that any row from position `first_position` on can see, but for those below the sequence's prefix. What lies
// between the two is never read: its blocks may be gone. (Positions ahead of the first key are negative: taken as they are,
// the subtraction of a window near 2^31 would wrap, and a walk begin outside the table.)
__device__ __forceinline__ int32_t window_start(const AttnParams &p, int32_t first_position) {
    return p.window > 0 ? max(0, max(0, first_position) - p.window + 1) : 0;
}

// 2^x for a difference of running maxima: a maximum of -inf (nothing seen yet) contributes nothing.
__device__ __forceinline__ float weight_of(float m, float reference) {
    return m == -INFINITY ? 0.f : exp2f(m - reference);
}

// The running join of partial results of one row: four of its output elements, relative to the maximum `top`.
struct Joined {
    float top = -INFINITY, sum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
};

// Joins n more parts in order; at(i) is part i's row index into `ml`, of [row][quads] float4 in `o`. Eight parts' loads are
// in flight together: one after another, each would wait for the L2 cache (0.5 us).
template <class At>
__device__ __forceinline__ void join_parts(Joined &j, int n, const float2 *ml, const float *o, int quads, int quad, At at) {
    constexpr int kAtOnce = 8;
    for (int i0 = 0; i0 < n; i0 += kAtOnce) {
        float2 part[kAtOnce];
        float4 x[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            part[k] = make_float2(-INFINITY, 0.f);
            x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (i0 + k < n) {
                const int64_t row = at(i0 + k);
                part[k] = __ldcg(&ml[row]);
                x[k] = __ldcg(reinterpret_cast<const float4 *>(o) + row * quads + quad);
            }
        }
        float top = j.top;
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) top = fmaxf(top, part[k].x);
        const float own = weight_of(j.top, top);
        j.top = top;
        j.sum *= own, j.o.x *= own, j.o.y *= own, j.o.z *= own, j.o.w *= own;
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const float f = weight_of(part[k].x, top);
            j.sum += f * part[k].y;
            j.o.x += f * x[k].x, j.o.y += f * x[k].y, j.o.z += f * x[k].z, j.o.w += f * x[k].w;
        }
    }
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float reciprocal_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <class T>
struct Pack2;
template <>
struct Pack2<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t of(float lo, float hi) {
        __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t *>(&v);
    }
};
template <>
struct Pack2<__half> {
    static __device__ __forceinline__ uint32_t of(float lo, float hi) {
        __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<uint32_t *>(&v);
    }
};

// Writes four elements of a finished row; one that sees nothing gets zeros.
template <class T>
__device__ __forceinline__ void write_row(const AttnParams &p, int token, int head, int quad, const Joined &j) {
    const float inverse = j.sum == 0.f ? 0.f : 1.f / j.sum;
    *reinterpret_cast<uint2 *>(p.out + (int64_t)token * p.out_token_stride + (int64_t)head * p.out_head_stride + quad * 8) =
        make_uint2(Pack2<T>::of(j.o.x * inverse, j.o.y * inverse), Pack2<T>::of(j.o.z * inverse, j.o.w * inverse));
}

}  // namespace kvx
