// Norm, rotation by position and the paged append of a step's rows, in one pass (kvx_rotate_store).
//
// Mathematics. A row x of a head becomes, in 32 bits and rounded once at the end,
//     y_i = x_i * rsqrt(mean_{j < norm_dim} x_j^2 + eps) * weight_i          for i < norm_dim, else y_i = x_i
// and each pair (a, b) of its rotary_dim elements from rotary_first on, with the angle's cos c and sin s of the
// row's position,
//     (a, b) -> (a c - b s, b c + a s).
// Pairs are (2p, 2p + 1) when interleaved, else (p, p + rotary_dim / 2). Queries go to query_out; keys (or latents)
// and values to their slots in every destination, as kvx_store places them. A key head is 1 norm, 1 rotation and
// 1 write instead of three passes over it.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "kvx_internal.cuh"

namespace {

using namespace kvx;

struct Rows {
    uint64_t base;
    int64_t token_stride, head_stride;  // bytes
    const void *weight;
    int32_t heads, dim, norm_dim, rotary_first;
};

struct RotateParams {
    Rows query, key, value;
    uint64_t out;
    int64_t out_token_stride, out_head_stride;  // bytes
    const float *table;                         // [num_positions][rotary_dim]: cos of every pair, then sin
    const void *positions;
    int32_t num_positions, rotary_dim, interleaved, position_bytes, num_tokens;
    float eps;
    int32_t n_dests, peers_only;
    int32_t *status, *error_word;
    StoreDest dests[kMaxStoreDests];
};

__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float x) {
    return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_float(float x) {
    return __float2half_rn(x);
}

__device__ __forceinline__ int64_t load_index(const void *p, int32_t bytes, int64_t i) {
    return bytes == 8 ? static_cast<const int64_t *>(p)[i] : static_cast<const int32_t *>(p)[i];
}

// Where destination d keeps token `token`'s row, as a byte offset from its caches' block 0; -1: nowhere (padding, a
// block its map leaves out, or a slot past the cache, which is flagged). `first` is the token's slot in destination 0.
__device__ __forceinline__ int64_t dest_offset(const RotateParams &p, int d, int64_t token, int64_t first) {
    const StoreDest &dst = p.dests[d];
    int64_t slot = first;
    if (d > 0 && !dst.block_map) slot = load_index(dst.slots, dst.slot_bytes, token);
    if (slot < 0) return -1;
    if (dst.block_map) {
        const int64_t b = slot / dst.block_size;
        if (b >= dst.block_map_len) {
            flag_error(p.error_word, p.status, kErrPastCache);
            return -1;
        }
        const int32_t mapped = dst.block_map[b];
        if (mapped < 0) return -1;
        slot = (int64_t)mapped * dst.block_size + (slot - b * dst.block_size);
    }
    if (slot >= (int64_t)dst.num_blocks * dst.block_size) {
        flag_error(p.error_word, p.status, kErrPastCache);
        return -1;
    }
    const uint32_t s = (uint32_t)slot;  // below 2^31: num_blocks * block_size is
    const uint32_t block = dst.block_shift >= 0 ? s >> dst.block_shift : s / (uint32_t)dst.block_size;
    const uint32_t in_block = s - block * (uint32_t)dst.block_size;
    return (int64_t)block * dst.block_stride + (int64_t)in_block * dst.token_stride;
}

// The table's row for token `token`; a position outside the table is flagged and read as its nearest row.
__device__ __forceinline__ const float *angles(const RotateParams &p, int64_t token, bool padding) {
    int64_t position = load_index(p.positions, p.position_bytes, token);
    if (position < 0 || position >= p.num_positions) {
        if (!padding) flag_error(p.error_word, p.status, kErrPosition);  // a padding row's position means nothing
        position = position < 0 ? 0 : p.num_positions - 1;
    }
    return p.table + position * p.rotary_dim;
}

constexpr int kAnyThreads = 256;

// The form for any width, stride and alignment: one warp per row, one element per lane at a time. Rows are read twice
// (the second time from L1): once for the sum of squares, once for the result.
template <class T>
__global__ void __launch_bounds__(kAnyThreads) rotate_store_any(const __grid_constant__ RotateParams p) {
    launch_dependents();
    wait_prerequisites();
    const int lane = threadIdx.x & 31;
    const int64_t rows_per_token = p.query.heads + p.key.heads + p.value.heads;
    const int64_t n = rows_per_token * p.num_tokens;
    for (int64_t w = (int64_t)blockIdx.x * (kAnyThreads / 32) + threadIdx.x / 32; w < n;
         w += (int64_t)gridDim.x * (kAnyThreads / 32)) {
        const int64_t token = w / rows_per_token;
        int head = (int)(w - token * rows_per_token);
        const int kind = head < p.query.heads ? 0 : head < p.query.heads + p.key.heads ? 1 : 2;
        const Rows &rows = kind == 0 ? p.query : kind == 1 ? p.key : p.value;
        head -= kind == 0 ? 0 : kind == 1 ? p.query.heads : p.query.heads + p.key.heads;
        const T *in = reinterpret_cast<const T *>(rows.base + token * rows.token_stride + head * rows.head_stride);
        const T *weight = static_cast<const T *>(rows.weight);
        const int64_t slot = load_index(p.dests[0].slots, p.dests[0].slot_bytes, token);

        T *to[kMaxStoreDests];
        int n_to = 0;
        if (kind == 0) {
            to[n_to++] = reinterpret_cast<T *>(p.out + token * p.out_token_stride + head * p.out_head_stride);
        } else {
            for (int d = p.peers_only; d < p.n_dests; ++d) {
                const StoreDest &dst = p.dests[d];
                if (head < dst.src_first_head || head >= dst.src_first_head + dst.num_heads) continue;
                const int64_t at = dest_offset(p, d, token, slot);
                if (at < 0) continue;
                to[n_to++] = reinterpret_cast<T *>((kind == 1 ? dst.k : dst.v) + at +
                                                   (int64_t)(head - dst.src_first_head + dst.dst_first_head) *
                                                       dst.head_stride);
            }
            if (n_to == 0) continue;  // the same for all lanes
        }

        float scale = 1.f;
        if (rows.norm_dim > 0) {
            float sum = 0.f;
            for (int i = lane; i < rows.norm_dim; i += 32) {
                const float x = to_float(in[i]);
                sum += x * x;
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
            scale = rsqrtf(sum / (float)rows.norm_dim + p.eps);
        }
        auto value_at = [&](int i) {
            const float x = to_float(in[i]);
            return i < rows.norm_dim ? x * scale * to_float(weight[i]) : x;
        };
        const int rotary = kind == 2 ? 0 : p.rotary_dim, half = rotary / 2;
        if (half > 0) {
            const float *angle = angles(p, token, slot < 0);
            for (int pair = lane; pair < half; pair += 32) {
                const int i = rows.rotary_first + (p.interleaved ? 2 * pair : pair);
                const int j = p.interleaved ? i + 1 : i + half;
                const float a = value_at(i), b = value_at(j), c = angle[pair], s = angle[half + pair];
                const T x = from_float<T>(a * c - b * s), y = from_float<T>(b * c + a * s);
                for (int t = 0; t < n_to; ++t) to[t][i] = x, to[t][j] = y;
            }
        }
        for (int i = lane; i < rows.dim - rotary; i += 32) {
            const int at = i < rows.rotary_first ? i : i + rotary;
            const T x = from_float<T>(value_at(at));
            for (int t = 0; t < n_to; ++t) to[t][at] = x;
        }
    }
}

int check_rows(const char *what, const kvx_rotate_rows &r, int rotary_dim) {
    if (r.num_heads < 0 || r.dim < 1 || r.norm_dim < 0 || r.norm_dim > r.dim)
        return fail(KVX_ERR_INVALID, "%s: bad row shape: %d heads of %d, %d normed", what, r.num_heads, r.dim,
                    r.norm_dim);
    if (!r.rows) return fail(KVX_ERR_INVALID, "%s: null rows", what);
    if (r.norm_dim > 0 && !r.weight) return fail(KVX_ERR_INVALID, "%s: a norm needs its weight", what);
    if (r.rotary_first < 0 || (int64_t)r.rotary_first + rotary_dim > r.dim)
        return fail(KVX_ERR_INVALID, "%s: rotated elements [%d, +%d) of %d", what, r.rotary_first, rotary_dim, r.dim);
    return KVX_OK;
}

Rows rows_of(const kvx_rotate_rows &r) {
    return Rows{(uint64_t)(uintptr_t)r.rows, r.token_stride, r.head_stride, r.weight,
                r.num_heads, r.dim, r.norm_dim, r.rotary_first};
}

}  // namespace

extern "C" int kvx_rotate_store(const kvx_rotate_args *args, const kvx_store_dest *dests, int n_dests, int32_t *status,
                                int flags, void *stream) {
    Range range("kvx_rotate_store");
    if (!args || !dests) return fail(KVX_ERR_INVALID, "null arguments or destinations");
    const kvx_rotate_args &a = *args;
    if (a.num_tokens < 0) return fail(KVX_ERR_INVALID, "%d tokens", a.num_tokens);
    if (a.dtype != KVX_BF16 && a.dtype != KVX_FP16) return fail(KVX_ERR_INVALID, "unknown element type %d", a.dtype);
    if (a.rotary_dim < 0 || a.rotary_dim % 2 != 0)
        return fail(KVX_ERR_INVALID, "rotary_dim %d is not an even number", a.rotary_dim);
    if (a.rotary_dim > 0 && a.num_tokens > 0 &&
        (!a.table || !a.positions || a.num_positions < 1 || (a.position_bytes != 4 && a.position_bytes != 8)))
        return fail(KVX_ERR_INVALID, "a rotation needs a table of one position at least, and 4- or 8-byte positions");
    const bool has_query = a.query.num_heads > 0, has_value = a.value.num_heads > 0;
    RotateParams p{};
    if (a.num_tokens > 0) {
        if (has_query) {
            if (int rc = check_rows("queries", a.query, a.rotary_dim)) return rc;
            if (!a.query_out) return fail(KVX_ERR_INVALID, "null query output");
            p.query = rows_of(a.query);
        }
        if (a.key.num_heads < 1) return fail(KVX_ERR_INVALID, "%d key heads", a.key.num_heads);
        if (int rc = check_rows("keys", a.key, a.rotary_dim)) return rc;
        p.key = rows_of(a.key);
        if (has_value) {
            if (int rc = check_rows("values", a.value, 0)) return rc;
            if (a.value.num_heads != a.key.num_heads || a.value.dim != a.key.dim || a.value.norm_dim != 0)
                return fail(KVX_ERR_INVALID, "values are plain rows of the keys' shape");
            p.value = rows_of(a.value);
        }
    }
    uint64_t align_bits = 0;
    if (int rc = fill_dests(dests, n_dests, a.num_tokens, a.key.num_heads, has_value, p.dests, &align_bits)) return rc;
    if (a.num_tokens == 0) return KVX_OK;
    if (!p.dests[0].slots) return fail(KVX_ERR_INVALID, "destination 0: null slots");
    p.out = (uint64_t)(uintptr_t)a.query_out;
    p.out_token_stride = a.out_token_stride;
    p.out_head_stride = a.out_head_stride;
    p.table = a.table;
    p.positions = a.positions;
    p.num_positions = a.num_positions;
    p.rotary_dim = a.rotary_dim;
    p.interleaved = a.interleaved;
    p.position_bytes = a.position_bytes;
    p.num_tokens = a.num_tokens;
    p.eps = a.eps;
    p.n_dests = n_dests;
    p.peers_only = (flags & KVX_STORE_PEERS_ONLY) ? 1 : 0;
    p.status = status;
    Device device;
    if (int rc = current_device(&device)) return rc;
    p.error_word = device.error_word;
    const int sm_budget = (flags >> 24) & 0xff;
    const int sms = sm_budget > 0 && sm_budget < device.sms ? sm_budget : device.sms;

    cudaLaunchConfig_t cfg = {};
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = (flags & KVX_STORE_SERIAL) ? 0 : 1;
    const int64_t rows = (int64_t)(p.query.heads + p.key.heads + p.value.heads) * p.num_tokens;
    const int64_t warps = kAnyThreads / 32;
    cfg.gridDim = dim3((unsigned)std::min<int64_t>((rows + warps - 1) / warps, (int64_t)sms * 8));
    cfg.blockDim = dim3(kAnyThreads);
    KVX_CUDA(cudaLaunchKernelEx(&cfg, a.dtype == KVX_BF16 ? rotate_store_any<__nv_bfloat16> : rotate_store_any<__half>,
                                p));
    count_launch();
    return KVX_OK;
}
