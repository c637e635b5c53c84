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

// ---- the form for the usual heads: 64, 128 or 256 wide, aligned rows, a rotary_dim that is a multiple of 8
//
// A row takes D / 8 lanes, each with the two 4-element pieces that rotate into each other (elements p and
// p + rotary_dim / 2, or 8 neighbours when interleaved or not rotated), so that no element changes lanes; the sum of
// squares is the one exchange. A warp takes PASSES x (256 / D) rows of one token, all their loads in flight at once, and
// reads the token's angles, slot and norm weights once for them. Bound by HBM: a step's rows in and out, once.

constexpr int kFastThreads = 256;
// One resident wave of 4 CTAs per SM at 64 registers. 8192 tokens of 32 + 8 + 8 heads of 128: 37.1 us (5.55 TB/s); with
// twice as many CTAs 38.5, with a CTA for every 8 units 47; 5 resident CTAs (48 registers) 43.2, 6 with half the loads in
// flight 54.7.
constexpr int kFastCtas = 4;

__device__ __forceinline__ float2 unpack(uint32_t bits, __nv_bfloat16) {
    return make_float2(__uint_as_float(bits << 16), __uint_as_float(bits & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack(uint32_t bits, __half) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&bits));
}
__device__ __forceinline__ uint32_t pack(float x, float y, __nv_bfloat16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t pack(float x, float y, __half) {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&v);
}

template <class T>
struct Piece {  // four elements
    uint2 bits;
    __device__ __forceinline__ void get(float2 (&x)[2]) const {
        x[0] = unpack(bits.x, T());
        x[1] = unpack(bits.y, T());
    }
    __device__ __forceinline__ void set(const float2 (&x)[2]) {
        bits = make_uint2(pack(x[0].x, x[0].y, T()), pack(x[1].x, x[1].y, T()));
    }
};

// Rows may be the output's own (queries rotated in place), so they are read as ordinary memory, past L1.
template <class T>
__device__ __forceinline__ Piece<T> load_piece(uint64_t at) {
    Piece<T> p;
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(p.bits.x), "=r"(p.bits.y) : "l"(at));
    return p;
}
template <class T>
__device__ __forceinline__ void store_piece(uint64_t at, const Piece<T> &p) {
    *reinterpret_cast<uint2 *>(at) = p.bits;
}

// A lane's place in a row, and its angles.
struct Place {
    int32_t a, b;  // first elements of its two pieces
    bool rotated;
};
template <bool INTERLEAVED>
__device__ __forceinline__ Place place_of(int lane_in_row, int rotary_dim) {
    Place p;
    p.rotated = 8 * lane_in_row < rotary_dim;
    const bool halves = !INTERLEAVED && p.rotated;
    p.a = halves ? 4 * lane_in_row : 8 * lane_in_row;
    p.b = halves ? rotary_dim / 2 + 4 * lane_in_row : 8 * lane_in_row + 4;
    return p;
}

// Turns the pairs of a and b by the angles whose cos and sin are c and s: two by two in one instruction where they lie in
// halves.
template <bool INTERLEAVED>
__device__ __forceinline__ void rotate(float2 (&a)[2], float2 (&b)[2], const float4 &c, const float4 &s) {
    if (INTERLEAVED) {
        auto turn = [](float2 &x, float cos, float sin) {
            x = make_float2(x.x * cos - x.y * sin, x.y * cos + x.x * sin);
        };
        turn(a[0], c.x, s.x);
        turn(a[1], c.y, s.y);
        turn(b[0], c.z, s.z);
        turn(b[1], c.w, s.w);
    } else {
        const float2 cos[2] = {make_float2(c.x, c.y), make_float2(c.z, c.w)};
        const float2 sin[2] = {make_float2(s.x, s.y), make_float2(s.z, s.w)};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 minus = make_float2(-sin[i].x, -sin[i].y), x = a[i];
            a[i] = fma2(b[i], minus, mul2(x, cos[i]));
            b[i] = fma2(x, sin[i], mul2(b[i], cos[i]));
        }
    }
}

__device__ __forceinline__ float squares(const float2 (&a)[2], const float2 (&b)[2]) {
    const float2 sum = fma2(b[1], b[1], fma2(b[0], b[0], fma2(a[1], a[1], mul2(a[0], a[0]))));
    return sum.x + sum.y;
}

// PASSES x (32 / LANES) rows of one token and one kind (0 queries, 1 keys, 2 values) from head `head0` on.
template <class T, int LANES, int PASSES, bool INTERLEAVED>
__device__ __forceinline__ void rotate_rows(const RotateParams &p, const Rows &rows, int kind, int64_t token, int head0,
                                            const Place &place) {
    constexpr int kAtOnce = 32 / LANES;
    const int lane = threadIdx.x & 31, lane_in_row = lane % LANES;
    const int first = head0 + lane / LANES;
    const uint64_t in = rows.base + token * rows.token_stride + first * rows.head_stride;
    Piece<T> x[PASSES], y[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        x[i].bits = y[i].bits = make_uint2(0, 0);
        if (first + i * kAtOnce < rows.heads) {
            const uint64_t at = in + i * kAtOnce * rows.head_stride;
            x[i] = load_piece<T>(at + place.a * sizeof(T));
            y[i] = load_piece<T>(at + place.b * sizeof(T));
        }
    }
    const int64_t slot = load_index(p.dests[0].slots, p.dests[0].slot_bytes, token);
    if (kind < 2) {
        float4 cos4, sin4;
        Piece<T> weight[2];
        if (place.rotated) {
            const float *angle = angles(p, token, slot < 0);
            cos4 = __ldg(reinterpret_cast<const float4 *>(angle) + lane_in_row);
            sin4 = __ldg(reinterpret_cast<const float4 *>(angle + p.rotary_dim / 2) + lane_in_row);
        }
        const bool normed = rows.norm_dim > 0;
        if (normed) {
            weight[0] = load_piece<T>((uint64_t)rows.weight + place.a * sizeof(T));
            weight[1] = load_piece<T>((uint64_t)rows.weight + place.b * sizeof(T));
        }
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            float2 a[2], b[2];
            x[i].get(a);
            y[i].get(b);
            if (normed) {
                float sum = squares(a, b);
#pragma unroll
                for (int o = LANES / 2; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
                const float scale = rsqrtf(sum * (1.f / (LANES * 8)) + p.eps);
                const float2 scales = make_float2(scale, scale);
                float2 w[2], v[2];
                weight[0].get(w);
                weight[1].get(v);
#pragma unroll
                for (int e = 0; e < 2; ++e) a[e] = mul2(mul2(a[e], scales), w[e]), b[e] = mul2(mul2(b[e], scales), v[e]);
            }
            if (place.rotated) rotate<INTERLEAVED>(a, b, cos4, sin4);
            x[i].set(a);
            y[i].set(b);
        }
    }
    auto store = [&](uint64_t to, int64_t head_stride, int from_head, int heads) {  // `to`: head 0's row
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int head = first + i * kAtOnce;
            if (head < from_head || head >= heads) continue;
            const uint64_t at = to + head * head_stride;
            store_piece<T>(at + place.a * sizeof(T), x[i]);
            store_piece<T>(at + place.b * sizeof(T), y[i]);
        }
    };
    if (kind == 0) {
        store(p.out + token * p.out_token_stride, p.out_head_stride, 0, rows.heads);
        return;
    }
    for (int d = p.peers_only; d < p.n_dests; ++d) {
        const StoreDest &dst = p.dests[d];
        const int64_t at = dest_offset(p, d, token, slot);
        if (at < 0) continue;
        store((kind == 1 ? dst.k : dst.v) + at + (int64_t)(dst.dst_first_head - dst.src_first_head) * dst.head_stride,
              dst.head_stride, dst.src_first_head, min(rows.heads, dst.src_first_head + dst.num_heads));
    }
}

template <class T, int LANES, int PASSES, bool INTERLEAVED>
__global__ void __launch_bounds__(kFastThreads, kFastCtas) rotate_store_fast(const __grid_constant__ RotateParams p) {
    launch_dependents();
    const Place place = place_of<INTERLEAVED>((threadIdx.x & 31) % LANES, p.rotary_dim);
    constexpr int kRows = PASSES * (32 / LANES);
    const uint32_t q_units = (p.query.heads + kRows - 1) / kRows, kv_units = (p.key.heads + kRows - 1) / kRows;
    const uint32_t per_token = q_units + 2 * kv_units, n = per_token * (uint32_t)p.num_tokens;
    wait_prerequisites();
    for (uint32_t w = blockIdx.x * (kFastThreads / 32) + threadIdx.x / 32; w < n; w += gridDim.x * (kFastThreads / 32)) {
        const uint32_t token = w / per_token, unit = w - token * per_token;
        const int kind = unit < q_units ? 0 : unit < q_units + kv_units ? 1 : 2;  // the same for a warp
        const Rows &rows = kind == 0 ? p.query : kind == 1 ? p.key : p.value;
        const int head0 = (unit - (kind == 0 ? 0 : kind == 1 ? q_units : q_units + kv_units)) * kRows;
        rotate_rows<T, LANES, PASSES, INTERLEAVED>(p, rows, kind, token, head0, place);
    }
}

// 8191 latents of 512 + 64 with 16 query heads (54.7 MB) take 11.1 us, 4.9 TB/s: a launch this short is mostly ramp.
//
// Latent rows of 256 x CHUNKS normed elements (or plain ones) and 64 rotated ones, a warp each, and the queries' rotated
// parts, 64 wide, 16 rows a warp.
template <class T, int CHUNKS, bool INTERLEAVED>
__global__ void __launch_bounds__(kFastThreads) rotate_latents_fast(const __grid_constant__ RotateParams p) {
    launch_dependents();
    const int lane = threadIdx.x & 31;
    constexpr int kLanes = 8, kPasses = 4, kRows = kPasses * (32 / kLanes), kRank = 256 * CHUNKS;
    const Place place = place_of<INTERLEAVED>(lane % kLanes, 64);
    const uint32_t per_token = 1 + (p.query.heads + kRows - 1) / kRows, n = per_token * (uint32_t)p.num_tokens;
    wait_prerequisites();
    for (uint32_t w = blockIdx.x * (kFastThreads / 32) + threadIdx.x / 32; w < n; w += gridDim.x * (kFastThreads / 32)) {
        const uint32_t token = w / per_token, item = w - token * per_token;
        if (item > 0) {
            rotate_rows<T, kLanes, kPasses, INTERLEAVED>(p, p.query, 0, token, (item - 1) * kRows, place);
            continue;
        }
        const int64_t slot = load_index(p.dests[0].slots, p.dests[0].slot_bytes, token);
        const float *angle = angles(p, token, slot < 0);
        const uint64_t row = p.key.base + (int64_t)token * p.key.token_stride;
        Piece<T> c[CHUNKS][2], x, y;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) c[k][h] = load_piece<T>(row + ((k * 64 + h * 32 + lane) * 4) * sizeof(T));
        if (lane < kLanes) {
            x = load_piece<T>(row + (kRank + place.a) * sizeof(T));
            y = load_piece<T>(row + (kRank + place.b) * sizeof(T));
        }
        if (p.key.norm_dim > 0) {
            Piece<T> weight[CHUNKS][2];
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    weight[k][h] = load_piece<T>((uint64_t)p.key.weight + ((k * 64 + h * 32 + lane) * 4) * sizeof(T));
                    float2 v[2];
                    c[k][h].get(v);
                    const float2 two = fma2(v[1], v[1], mul2(v[0], v[0]));
                    sum += two.x + two.y;
                }
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
            const float scale = rsqrtf(sum * (1.f / kRank) + p.eps);
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float2 v[2], m[2];
                    c[k][h].get(v);
                    weight[k][h].get(m);
#pragma unroll
                    for (int e = 0; e < 2; ++e) v[e] = mul2(mul2(v[e], make_float2(scale, scale)), m[e]);
                    c[k][h].set(v);
                }
        }
        if (lane < kLanes) {
            float2 a[2], b[2];
            x.get(a);
            y.get(b);
            rotate<INTERLEAVED>(a, b, __ldg(reinterpret_cast<const float4 *>(angle) + lane),
                                __ldg(reinterpret_cast<const float4 *>(angle + 32) + lane));
            x.set(a);
            y.set(b);
        }
        for (int d = p.peers_only; d < p.n_dests; ++d) {
            const StoreDest &dst = p.dests[d];
            if (dst.num_heads < 1) continue;
            const int64_t at = dest_offset(p, d, token, slot);
            if (at < 0) continue;
            const uint64_t to = dst.k + at + (int64_t)dst.dst_first_head * dst.head_stride;
#pragma unroll
            for (int k = 0; k < CHUNKS; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) store_piece<T>(to + ((k * 64 + h * 32 + lane) * 4) * sizeof(T), c[k][h]);
            if (lane < kLanes) {
                store_piece<T>(to + (kRank + place.a) * sizeof(T), x);
                store_piece<T>(to + (kRank + place.b) * sizeof(T), y);
            }
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

// One warp per unit of work, `ctas_per_sm` CTAs at most: each sweeps its share.
int launch(void (*kernel)(RotateParams), const RotateParams &p, cudaLaunchConfig_t cfg, int64_t units, int sms,
           int ctas_per_sm) {
    static_assert(kFastThreads == kAnyThreads, "one block size");
    constexpr int kWarps = kFastThreads / 32;
    cfg.gridDim = dim3((unsigned)std::min<int64_t>((units + kWarps - 1) / kWarps, (int64_t)sms * ctas_per_sm));
    cfg.blockDim = dim3(kFastThreads);
    KVX_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    count_launch();
    return KVX_OK;
}

// Warps a token's rows take at `at_once` rows a unit.
int units_of(const RotateParams &p, int at_once) {
    return (p.query.heads + at_once - 1) / at_once + 2 * ((p.key.heads + at_once - 1) / at_once);
}

template <class T, int LANES, int PASSES>
int launch_rows(const RotateParams &p, const cudaLaunchConfig_t &cfg, int sms) {
    return launch(p.interleaved ? rotate_store_fast<T, LANES, PASSES, true> : rotate_store_fast<T, LANES, PASSES, false>, p,
                  cfg, (int64_t)units_of(p, PASSES * (32 / LANES)) * p.num_tokens, sms, kFastCtas);
}

template <class T, int LANES>
int launch_lanes(const RotateParams &p, const cudaLaunchConfig_t &cfg, int sms) {
    // Four passes of rows a warp keep the most loads in flight; fewer where they leave warps with too little to do:
    // heads that do not fill them, or too few tokens to give every scheduler a warp.
    const int rows = p.query.heads + p.key.heads + p.value.heads, at_once = 32 / LANES;
    auto fits = [&](int passes) {
        const int units = units_of(p, passes * at_once);
        return rows * 4 >= units * passes * at_once * 3 && (int64_t)units * p.num_tokens >= (int64_t)sms * 4;
    };
    if (fits(4)) return launch_rows<T, LANES, 4>(p, cfg, sms);
    if (fits(2)) return launch_rows<T, LANES, 2>(p, cfg, sms);
    return launch_rows<T, LANES, 1>(p, cfg, sms);
}

template <class T>
int launch_fast(const RotateParams &p, const cudaLaunchConfig_t &cfg, int sms) {
    return p.key.dim == 64    ? launch_lanes<T, 8>(p, cfg, sms)
           : p.key.dim == 128 ? launch_lanes<T, 16>(p, cfg, sms)
                              : launch_lanes<T, 32>(p, cfg, sms);
}

template <class T, int CHUNKS>
int launch_chunks(const RotateParams &p, const cudaLaunchConfig_t &cfg, int sms) {
    return launch(p.interleaved ? rotate_latents_fast<T, CHUNKS, true> : rotate_latents_fast<T, CHUNKS, false>, p, cfg,
                  (int64_t)(1 + (p.query.heads + 15) / 16) * p.num_tokens, sms, 8);
}

template <class T>
int launch_latents(const RotateParams &p, const cudaLaunchConfig_t &cfg, int sms, int chunks) {
    return chunks == 1   ? launch_chunks<T, 1>(p, cfg, sms)
           : chunks == 2 ? launch_chunks<T, 2>(p, cfg, sms)
           : chunks == 3 ? launch_chunks<T, 3>(p, cfg, sms)
                         : launch_chunks<T, 4>(p, cfg, sms);
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
    // The push half of a store leaves the queries to the local half, which may have rotated them in place.
    const bool has_query = a.query.num_heads > 0 && !(flags & KVX_STORE_PEERS_ONLY), has_value = a.value.num_heads > 0;
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
    // The vector forms move 8 bytes at a time; what they do not take goes row by row, element by element.
    const int heads = p.query.heads + p.key.heads + p.value.heads;
    align_bits |= p.query.base | p.key.base | p.value.base | (uint64_t)p.query.token_stride |
                  (uint64_t)p.query.head_stride | (uint64_t)p.key.token_stride | (uint64_t)p.key.head_stride |
                  (uint64_t)p.value.token_stride | (uint64_t)p.value.head_stride | (uint64_t)(uintptr_t)p.query.weight |
                  (uint64_t)(uintptr_t)p.key.weight | (has_query ? p.out : 0) |
                  (has_query ? (uint64_t)p.out_token_stride | (uint64_t)p.out_head_stride : 0);
    const bool aligned = align_bits % 8 == 0 && (uint64_t)(uintptr_t)p.table % 16 == 0 && p.rotary_dim % 8 == 0 &&
                         (int64_t)heads * p.num_tokens < (int64_t)1 << 31;
    const int dim = p.key.dim;
    const bool plain = p.key.rotary_first == 0 && (p.key.norm_dim == 0 || p.key.norm_dim == dim);
    const bool queries_plain = !has_query || (p.query.dim == dim && p.query.rotary_first == 0 &&
                                              (p.query.norm_dim == 0 || p.query.norm_dim == dim));
    const bool bf16 = a.dtype == KVX_BF16;
    if (aligned && plain && queries_plain && has_value && (dim == 64 || dim == 128 || dim == 256))
        return bf16 ? launch_fast<__nv_bfloat16>(p, cfg, sms) : launch_fast<__half>(p, cfg, sms);
    const int rank = dim - 64;
    if (aligned && !has_value && p.rotary_dim == 64 && p.key.heads == 1 && p.key.rotary_first == rank &&
        (p.key.norm_dim == 0 || p.key.norm_dim == rank) && rank >= 256 && rank <= 1024 && rank % 256 == 0 &&
        (!has_query || (p.query.dim == 64 && p.query.rotary_first == 0 && p.query.norm_dim == 0)))
        return bf16 ? launch_latents<__nv_bfloat16>(p, cfg, sms, rank / 256) : launch_latents<__half>(p, cfg, sms, rank / 256);
    return launch(bf16 ? rotate_store_any<__nv_bfloat16> : rotate_store_any<__half>, p, cfg,
                  (int64_t)heads * p.num_tokens, sms, 8);
}
