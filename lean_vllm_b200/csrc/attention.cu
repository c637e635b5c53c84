// Attention over the paged cache (kvx_attention).
//
// Mathematics. For a query row at position i, over the keys j that its mask leaves,
//     s_j = cap(scale q.k_j) + slope (j - i),   o = sum_j 2^(t_j - m) v_j / sum_j 2^(t_j - m),   t_j = s_j log2(e)
// in one pass with the running maximum m and sum of the softmax. Scores, maxima, sums and the accumulated output are
// held in 32 bits; the weights 2^(t_j - m) are rounded to the cache's 16-bit type for the tensor cores' second product
// (each is below 2^0, so the rounding is relative, 2^-9 in bf16, and averages out over the keys).

#include <algorithm>

#include "attention.cuh"

namespace {

using namespace kvx;

// ------------------------------------------------------------------------------------------------ rows kernel
//
// attention_rows: up to 16 query rows of one KV head (its group of query heads x the sequence's query tokens) against
// a stretch of a sequence's keys: the form for single tokens, bound by reading the cache.
//
// Work. The rows of a KV head share its keys, so a (sequence, KV head, tile of 16 rows) group reads them once. Its
// keys are cut into tiles of 64 tokens; the tiles of all groups of all sequences, counted on the device from the
// lengths, are dealt out in equal contiguous runs to a grid of two CTAs per SM, whatever the lengths. A CTA's run
// covers whole groups and at most two partial ones; a partial group leaves (m, sum, o) in the workspace, and the CTA
// that brings the last part joins them in a fixed order (the result does not depend on which one that is).
//
// Inside a CTA each of the 4 warps takes its own 16 tokens of every tile with its own running maximum, sum and output,
// and loads them itself with cp.async into its own ring of 3 stages: no barrier until the group's end.

constexpr int kRowTile = 16;
constexpr int kRowWarps = 4;
constexpr int kRowThreads = kRowWarps * 32;
constexpr int kRowStages = 3;
constexpr int kWarpTokens = 16;
constexpr int kTileTokens = kRowWarps * kWarpTokens;

template <int D>
constexpr int row_smem() {
    return kRowWarps * kRowStages * kWarpTokens * D * 2 * 2;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool valid) {
    const int bytes = valid ? 16 : 0;  // the rest is filled with zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

template <class T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t *a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A sequence's share of the launch's tiles.
struct RowWork {
    int32_t lo, row_tiles, tiles;  // first key, tiles of rows, tiles of keys per group
    __device__ __forceinline__ int64_t groups(const AttnParams &p) const { return (int64_t)row_tiles * p.kv_heads; }
};

__device__ __forceinline__ RowWork row_work(const AttnParams &p, const Sequence &q) {
    RowWork w;
    w.lo = first_seen(p, q, q.kv_len - q.q_len);
    w.row_tiles = (int32_t)(((int64_t)q.q_len * p.group + kRowTile - 1) / kRowTile);
    // An empty cache still gets one (empty) tile: its rows have to be written.
    w.tiles = max(1, (q.kv_len + kTileTokens - 1) / kTileTokens - w.lo / kTileTokens);
    return w;
}

__device__ __forceinline__ int64_t row_units(const AttnParams &p, int s) {
    if (blockIdx.x == 0 && (int64_t)p.kv_lens[s] > (int64_t)p.max_blocks * p.block_size)
        flag_error(p.error_word, p.status, kErrPastCache);
    const Sequence q = sequence_of(p, s);
    if ((int64_t)q.q_len * p.group > p.rows_limit) return 0;  // attention_tiles takes it
    const RowWork w = row_work(p, q);
    return w.groups(p) * w.tiles;
}

// The address of query row `row` (query token row / group, head row % group of KV head h) in a [token][head] tensor.
__device__ __forceinline__ uint64_t row_address(const AttnParams &p, uint64_t base, int64_t token_stride,
                                                int64_t head_stride, const Sequence &q, int h, int row) {
    const int token = row / p.group;
    return base + (int64_t)(q.q0 + token) * token_stride + (int64_t)(h * p.group + row - token * p.group) * head_stride;
}

template <class T, int D, bool MODS>
__global__ void __launch_bounds__(kRowThreads, 2) attention_rows(const __grid_constant__ AttnParams p) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int64_t scan[kRowWarps + 1];
    __shared__ int64_t found_start;
    __shared__ int found_sequence;
    __shared__ float2 warp_ml[kRowWarps][kRowTile];
    __shared__ int is_last;

    launch_dependents();
    // Behind a kernel that computes the shared prefix's part, only the joining below has to wait for it: that kernel
    // lets this one start after its own wait, so everything before it is complete.
    if (p.prefix_splits == 0) wait_prerequisites();

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    // ---- this CTA's run of tiles
    int64_t mine = 0;
    for (int s = tid; s < p.batch; s += kRowThreads) mine += row_units(p, s);
#pragma unroll
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(~0u, mine, o);
    if (lane == 0) scan[warp] = mine;
    __syncthreads();
    int64_t total = 0;
    for (int w = 0; w < kRowWarps; ++w) total += scan[w];
    const int64_t per_cta = (total + gridDim.x - 1) / gridDim.x;
    int64_t unit = (int64_t)blockIdx.x * per_cta;
    const int64_t unit_end = min(total, unit + per_cta);
    if (unit >= unit_end) {
        wait_prerequisites();
        return;
    }
    int64_t before = 0;  // tiles of the sequences looked at so far
    for (int s0 = 0;; s0 += kRowThreads) {
        const int s = s0 + tid;
        int64_t n = s < p.batch ? row_units(p, s) : 0, sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t up = __shfl_up_sync(~0u, sum, o);
            if (lane >= o) sum += up;
        }
        __syncthreads();
        if (lane == 31) scan[warp] = sum;
        __syncthreads();
        int64_t start = before + sum - n, chunk = 0;
        for (int w = 0; w < kRowWarps; ++w) {
            if (w < warp) start += scan[w];
            chunk += scan[w];
        }
        if (start <= unit && unit < start + n) {
            found_sequence = s;
            found_start = start;
        }
        before += chunk;
        if (unit < before) break;  // the same for all threads
    }
    __syncthreads();
    int s = found_sequence;
    int64_t s_start = found_start;

    constexpr int kChunks = D / 8;                 // 16-byte chunks of a row
    constexpr int kPerCopy = 32 / kChunks;         // tokens one warp-wide copy covers
    constexpr int kCopies = kWarpTokens / kPerCopy;
    constexpr int kStageBytes = kWarpTokens * D * 2;  // keys; as much again for values
    const uint32_t ring = smem_u32(smem) + warp * kRowStages * 2 * kStageBytes;
    float *my_o = reinterpret_cast<float *>(smem + warp * kRowStages * 2 * kStageBytes);  // once the ring is done with
    const float scale_log2 = p.scale * kLog2e;

    while (unit < unit_end) {
        const Sequence q = sequence_of(p, s);
        const RowWork work = row_work(p, q);
        const int64_t s_end = s_start + row_units(p, s);
        if (unit >= s_end) {
            s_start = s_end;
            ++s;
            continue;
        }
        const int64_t in_sequence = unit - s_start;
        const int64_t group_index = in_sequence / work.tiles;
        const int tile0 = (int)(in_sequence - group_index * work.tiles);
        const int h = (int)(group_index / work.row_tiles);
        const int row0 = (int)(group_index - (int64_t)h * work.row_tiles) * kRowTile;
        const int64_t group_start = s_start + group_index * work.tiles, group_end = group_start + work.tiles;
        const int n_tiles = (int)(min(unit_end, group_end) - unit);
        const int rows = min(kRowTile, q.q_len * p.group - row0);
        const int first_token = work.lo / kTileTokens * kTileTokens + tile0 * kTileTokens + warp * kWarpTokens;
        const int64_t head_offset = (int64_t)h * p.head_stride;

        // The byte offset of this lane's token (lanes 0-15) in stage i, or -1 where nothing is to be read.
        auto token_offset = [&](int i) -> int64_t {
            const int t = first_token + i * kTileTokens + lane;
            if (i >= n_tiles || lane >= kWarpTokens || t < work.lo || t >= q.kv_len) return -1;
            const int64_t at = token_at(p, s, t);
            return at < 0 ? -1 : at + head_offset;
        };
        auto load_stage = [&](int i, int64_t offset) {
            const uint32_t k_stage = ring + (i % kRowStages) * 2 * kStageBytes, v_stage = k_stage + kStageBytes;
#pragma unroll
            for (int c = 0; c < kCopies; ++c) {
                const int token = c * kPerCopy + lane / kChunks, chunk = lane % kChunks;
                const int64_t at = __shfl_sync(~0u, offset, token);
                const uint32_t to = token * D * 2 + ((chunk ^ (token & 7)) << 4);
                const int64_t from = at < 0 ? 0 : at + chunk * 16;
                cp_async16(k_stage + to, reinterpret_cast<const void *>(p.k_cache + from), at >= 0);
                cp_async16(v_stage + to, reinterpret_cast<const void *>(p.v_cache + from), at >= 0);
            }
        };
#pragma unroll
        for (int i = 0; i < kRowStages - 1; ++i) {
            if (i < n_tiles) load_stage(i, token_offset(i));
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        int64_t next_offset = token_offset(kRowStages - 1);

        // ---- queries, in the registers of the first product
        uint32_t qa[D / 16][4];
        int position[2], prefix[2];  // of rows lane / 4 and lane / 4 + 8
        float slope[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = lane / 4 + 8 * r;
            const bool valid = row < rows;
            const uint64_t at = valid ? row_address(p, p.query, p.q_token_stride, p.q_head_stride, q, h, row0 + row) : 0;
            position[r] = valid ? q.kv_len - q.q_len + (row0 + row) / p.group : -1;
            prefix[r] = valid ? q.prefix : 0;
            slope[r] = MODS && valid && p.slopes ? p.slopes[h * p.group + (row0 + row) % p.group] : 0.f;
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    qa[k][r + 2 * half] =
                        valid ? *reinterpret_cast<const uint32_t *>(at + (k * 16 + half * 8 + (lane & 3) * 2) * 2) : 0u;
        }
        // Every row of the tile sees the keys from see_lo up to see_hi: whole stages in there need no mask.
        const int first_position = q.kv_len - q.q_len + row0 / p.group;
        const int last_position = q.kv_len - q.q_len + (row0 + rows - 1) / p.group;
        const int see_lo = p.window > 0 ? max(work.lo, last_position - p.window + 1) : 0;
        const int see_hi = min(q.kv_len, first_position + 1);

        float m[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f}, o[D / 8][4];
#pragma unroll
        for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;

        for (int i = 0; i < n_tiles; ++i) {
            if (i + kRowStages - 1 < n_tiles) load_stage(i + kRowStages - 1, next_offset);
            asm volatile("cp.async.commit_group;" ::: "memory");
            next_offset = token_offset(i + kRowStages);
            asm volatile("cp.async.wait_group %0;" ::"n"(kRowStages - 1) : "memory");
            __syncwarp();
            const uint32_t k_stage = ring + (i % kRowStages) * 2 * kStageBytes, v_stage = k_stage + kStageBytes;
            const int t0 = first_token + i * kTileTokens;

            float c[2][4] = {};
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                uint32_t b[4];
                const int token = (lane & 7) + ((lane & 16) >> 1), chunk = 2 * k + ((lane >> 3) & 1);
                ldmatrix4(b, k_stage + token * D * 2 + ((chunk ^ (token & 7)) << 4));
                mma16816<T>(c[0], qa[k], b[0], b[1]);
                mma16816<T>(c[1], qa[k], b[2], b[3]);
            }
            const bool masked = t0 < see_lo || t0 + kWarpTokens > see_hi;
            float stage_max[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = e >> 1, t = t0 + n * 8 + (lane & 3) * 2 + (e & 1);
                    float x;
                    if (MODS) {
                        x = c[n][e] * p.scale;
                        if (p.softcap > 0.f) x = p.softcap * tanhf(x / p.softcap);
                        x = (x + slope[r] * (float)(t - position[r])) * kLog2e;
                    } else {
                        x = c[n][e] * scale_log2;
                    }
                    if (masked) {
                        const bool seen = t < q.kv_len && t >= work.lo &&
                                          ((t <= position[r] && (p.window <= 0 || t > position[r] - p.window)) ||
                                           t < prefix[r]);
                        x = seen ? x : -INFINITY;
                    }
                    c[n][e] = x;
                    stage_max[r] = fmaxf(stage_max[r], x);
                }
            float reference[2];
            bool grown = false;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                stage_max[r] = fmaxf(stage_max[r], __shfl_xor_sync(~0u, stage_max[r], 1));
                stage_max[r] = fmaxf(stage_max[r], __shfl_xor_sync(~0u, stage_max[r], 2));
                grown |= stage_max[r] > m[r];
            }
            if (__any_sync(~0u, grown)) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float now = fmaxf(m[r], stage_max[r]), factor = weight_of(m[r], now);
                    m[r] = now;
                    sum[r] *= factor;
#pragma unroll
                    for (int n = 0; n < D / 8; ++n) o[n][2 * r] *= factor, o[n][2 * r + 1] *= factor;
                }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) reference[r] = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    c[n][e] = exp2f(c[n][e] - reference[e >> 1]);
                    sum[e >> 1] += c[n][e];
                }
            const uint32_t pa[4] = {Pack2<T>::of(c[0][0], c[0][1]), Pack2<T>::of(c[0][2], c[0][3]),
                                    Pack2<T>::of(c[1][0], c[1][1]), Pack2<T>::of(c[1][2], c[1][3])};
#pragma unroll
            for (int n = 0; n < D / 8; n += 2) {
                uint32_t b[4];
                const int token = (lane & 7) + (lane & 8), chunk = n + (lane >> 4);
                ldmatrix4_trans(b, v_stage + token * D * 2 + ((chunk ^ (token & 7)) << 4));
                mma16816<T>(o[n], pa, b[0], b[1]);
                mma16816<T>(o[n + 1], pa, b[2], b[3]);
            }
            __syncwarp();
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();

        // ---- join the warps
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            sum[r] += __shfl_xor_sync(~0u, sum[r], 1);
            sum[r] += __shfl_xor_sync(~0u, sum[r], 2);
            const int row = lane / 4 + 8 * r;
            if ((lane & 3) == 0) warp_ml[warp][row] = make_float2(m[r], sum[r]);
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
                *reinterpret_cast<float2 *>(my_o + row * D + n * 8 + (lane & 3) * 2) =
                    make_float2(o[n][2 * r], o[n][2 * r + 1]);
        }
        __syncthreads();
        const bool whole = unit == group_start && n_tiles == work.tiles;
        const int c0 = (int)(group_start / per_cta), c1 = (int)((group_end - 1) / per_cta);
        const int slot = 2 * blockIdx.x + (unit == group_start ? 1 : 0);
        constexpr int kQuads = D / 4;
        constexpr int kWarpFloats = kRowStages * 2 * kStageBytes / 4;
        const float *all_o = reinterpret_cast<const float *>(smem);

        // Writes a row's four elements, after joining the parts over a shared prefix.
        auto finish = [&](int row, int quad, Joined j) {
            const int token = q.q0 + (row0 + row) / p.group, head = h * p.group + (row0 + row) % p.group;
            const int64_t at = (int64_t)token * p.q_heads + head, step = (int64_t)p.num_tokens * p.q_heads;
            join_parts(j, p.prefix_splits, p.split_ml, p.split_o, kQuads, quad, [&](int i) { return at + i * step; });
            const float inverse = j.sum == 0.f ? 0.f : 1.f / j.sum;  // a row that sees nothing gets zeros
            char *out = reinterpret_cast<char *>(p.out + (int64_t)token * p.out_token_stride +
                                                 (int64_t)head * p.out_head_stride) + quad * 8;
            *reinterpret_cast<uint2 *>(out) = make_uint2(Pack2<T>::of(j.o.x * inverse, j.o.y * inverse),
                                                         Pack2<T>::of(j.o.z * inverse, j.o.w * inverse));
        };

        if (whole && p.prefix_splits > 0) wait_prerequisites();
        for (int item = tid; item < rows * kQuads; item += kRowThreads) {
            const int row = item / kQuads, quad = item % kQuads;
            Joined j;
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) j.top = fmaxf(j.top, warp_ml[w][row].x);
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) {
                const float f = weight_of(warp_ml[w][row].x, j.top);
                const float4 x = reinterpret_cast<const float4 *>(all_o + w * kWarpFloats + row * D)[quad];
                j.sum += f * warp_ml[w][row].y;
                j.o.x += f * x.x, j.o.y += f * x.y, j.o.z += f * x.z, j.o.w += f * x.w;
            }
            if (whole) {
                finish(row, quad, j);
            } else {
                reinterpret_cast<float4 *>(p.partial_o)[(int64_t)(slot * kRowTile + row) * kQuads + quad] = j.o;
                if (quad == 0) p.partial_ml[slot * kRowTile + row] = make_float2(j.top, j.sum);
            }
        }
        if (!whole) {
            // ---- the group's last part to arrive joins all of them
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                is_last = atomicAdd(&p.counters[c0], 1) == c1 - c0;
                if (is_last) p.counters[c0] = 0;  // for the next launch
            }
            __syncthreads();
            if (is_last) {
                __threadfence();
                if (p.prefix_splits > 0) wait_prerequisites();
                for (int item = tid; item < rows * kQuads; item += kRowThreads) {
                    const int row = item / kQuads, quad = item % kQuads;
                    Joined j;
                    join_parts(j, c1 - c0 + 1, p.partial_ml, p.partial_o, kQuads, quad,
                               [&](int i) { return (int64_t)(2 * (c0 + i) + (i == 0)) * kRowTile + row; });
                    finish(row, quad, j);
                }
            }
        }
        __syncthreads();  // the ring and the joined values are free again
        unit += n_tiles;
    }
    wait_prerequisites();
}

// ------------------------------------------------------------------------------------------------ host side

constexpr size_t kRowPartials = (size_t)kMaxRowCtas * 2 * kRowTile;
constexpr size_t kMlBytes = sizeof(float2), kOutBytes = 128 * sizeof(float);
constexpr size_t kSplitAt = KVX_ATTENTION_ZEROED + kRowPartials * (kMlBytes + kOutBytes);
constexpr size_t kWorkspaceBytes = kSplitAt + kSplitRows * (kMlBytes + kOutBytes);
static_assert(kMaxRowCtas <= kTileCounter && (kTileCounter + 1) * sizeof(int32_t) <= KVX_ATTENTION_ZEROED, "counters");

template <class T, int D>
int launch_rows(const AttnParams &p, bool mods, const Device &device, cudaStream_t stream) {
    static AllowedSmem allowed[2];
    auto kernel = mods ? attention_rows<T, D, true> : attention_rows<T, D, false>;
    if (int rc = allowed[mods].allow(kernel, row_smem<D>(), device.index)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3((unsigned)std::min(2 * device.sms, kMaxRowCtas));
    cfg.blockDim = dim3(kRowThreads);
    cfg.dynamicSmemBytes = row_smem<D>();
    KVX_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    count_launch();
    return KVX_OK;
}

}  // namespace

extern "C" {

uint64_t kvx_attention_workspace_bytes(void) { return kWorkspaceBytes; }

int kvx_attention(const kvx_attention_args *args, int flags, void *stream) {
    Range range("kvx_attention");
    if (!args) return fail(KVX_ERR_INVALID, "null arguments");
    const kvx_attention_args &a = *args;
    if (a.num_tokens < 0 || a.batch < 0) return fail(KVX_ERR_INVALID, "%d tokens of %d sequences", a.num_tokens, a.batch);
    if (a.q_heads < 1 || a.kv_heads < 1 || a.q_heads % a.kv_heads != 0)
        return fail(KVX_ERR_INVALID, "%d query heads over %d KV heads", a.q_heads, a.kv_heads);
    if (a.head_dim != 64 && a.head_dim != 128) return fail(KVX_ERR_INVALID, "head_dim %d; 64 or 128", a.head_dim);
    if (a.dtype != KVX_BF16 && a.dtype != KVX_FP16) return fail(KVX_ERR_INVALID, "unknown element type %d", a.dtype);
    if (a.block_size < 1 || a.num_blocks < 0 || a.max_blocks < 0 || a.table_stride < 0 || a.shared_len < 0 ||
        a.shared_blocks < 0)
        return fail(KVX_ERR_INVALID, "bad block size, block count or table");
    if ((int64_t)a.max_blocks * a.block_size >= (int64_t)1 << 31 || a.shared_len >= 1 << 30)
        return fail(KVX_ERR_INVALID, "more than 2^31 tokens a sequence");
    if (a.window < 0 || !(a.softcap >= 0.f)) return fail(KVX_ERR_INVALID, "negative window or softcap");
    if ((int64_t)a.shared_blocks * a.block_size < a.shared_len)
        return fail(KVX_ERR_RANGE, "a shared prefix of %d tokens in %d blocks of %d", a.shared_len, a.shared_blocks,
                    a.block_size);
    if (a.shared_len > 0 && (a.window > 0 || a.prefix_lens))
        return fail(KVX_ERR_INVALID, "a shared prefix takes no window and no prefix_lens");
    if (a.num_tokens == 0 || a.batch == 0) return KVX_OK;
    if (!a.query || !a.out || !a.k_cache || !a.v_cache || !a.kv_lens || !a.workspace ||
        (a.max_blocks > 0 && !a.block_tables) || (a.shared_len > 0 && !a.shared_table))
        return fail(KVX_ERR_INVALID, "null pointer");
    if (!a.q_starts && a.num_tokens != a.batch)
        return fail(KVX_ERR_INVALID, "%d query tokens of %d sequences need q_starts", a.num_tokens, a.batch);
    const uint64_t bits = (uint64_t)(uintptr_t)a.query | (uint64_t)(uintptr_t)a.out | a.k_cache | a.v_cache |
                          (uint64_t)a.q_token_stride | (uint64_t)a.q_head_stride | (uint64_t)a.out_token_stride |
                          (uint64_t)a.out_head_stride | (uint64_t)a.block_stride | (uint64_t)a.token_stride |
                          (uint64_t)a.head_stride;
    if (bits % 16 != 0) return fail(KVX_ERR_INVALID, "queries, output and cache rows start on 16-byte boundaries");
    if ((uint64_t)(uintptr_t)a.workspace % 128 != 0) return fail(KVX_ERR_INVALID, "the workspace starts on 128 bytes");

    Device device;
    if (int rc = current_device(&device)) return rc;
    AttnParams p{};
    p.query = (uint64_t)(uintptr_t)a.query;
    p.out = (uint64_t)(uintptr_t)a.out;
    p.k_cache = a.k_cache;
    p.v_cache = a.v_cache;
    p.q_token_stride = a.q_token_stride;
    p.q_head_stride = a.q_head_stride;
    p.out_token_stride = a.out_token_stride;
    p.out_head_stride = a.out_head_stride;
    p.block_stride = a.block_stride;
    p.token_stride = a.token_stride;
    p.head_stride = a.head_stride;
    p.block_tables = a.block_tables;
    p.kv_lens = a.kv_lens;
    p.q_starts = a.q_starts;
    p.prefix_lens = a.prefix_lens;
    p.slopes = a.slopes;
    p.table_stride = a.table_stride;
    p.block_size = a.block_size;
    p.block_shift = -1;
    for (int k = 0; k < 31; ++k)
        if (a.block_size == (1 << k)) p.block_shift = k;
    p.num_blocks = a.num_blocks;
    p.max_blocks = a.max_blocks;
    p.batch = a.batch;
    p.num_tokens = a.num_tokens;
    p.q_heads = a.q_heads;
    p.kv_heads = a.kv_heads;
    p.group = a.q_heads / a.kv_heads;
    p.window = a.window;
    p.scale = a.scale;
    p.softcap = a.softcap;
    p.status = a.status;
    p.error_word = device.error_word;
    unsigned char *work = static_cast<unsigned char *>(a.workspace);
    p.counters = reinterpret_cast<int32_t *>(work);
    p.partial_ml = reinterpret_cast<float2 *>(work + KVX_ATTENTION_ZEROED);
    p.partial_o = reinterpret_cast<float *>(work + KVX_ATTENTION_ZEROED + kRowPartials * kMlBytes);
    p.split_ml = reinterpret_cast<float2 *>(work + kSplitAt);
    p.split_o = reinterpret_cast<float *>(work + kSplitAt + kSplitRows * kMlBytes);
    p.shared_table = a.shared_table;
    p.shared_len = a.shared_len;
    p.rows_limit = INT32_MAX;
    const bool mods = a.softcap > 0.f || a.slopes || !(a.scale > 0.f);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    auto rows_kernel = [&]() {
        if (a.head_dim == 128)
            return a.dtype == KVX_BF16 ? launch_rows<__nv_bfloat16, 128>(p, mods, device, s)
                                       : launch_rows<__half, 128>(p, mods, device, s);
        return a.dtype == KVX_BF16 ? launch_rows<__nv_bfloat16, 64>(p, mods, device, s)
                                   : launch_rows<__half, 64>(p, mods, device, s);
    };

    // ---- which kernel takes what
    const int64_t q_rows = (int64_t)std::max(a.max_q_len, 1) * p.group;  // of the longest sequence and one KV head
    const int64_t all_rows = (int64_t)a.num_tokens * p.group;
    // Splits of the keys that fill the device with one CTA per SM, two tiles of keys each at least, as many as the
    // workspace has room for.
    auto splits_for = [&](int64_t row_tiles, int64_t keys) {
        const int64_t fill = device.sms / std::max<int64_t>(1, row_tiles * a.kv_heads);
        const int64_t tiles = (keys + kTileKeys - 1) / kTileKeys;
        return (int)std::max<int64_t>(
            1, std::min({fill, (tiles + 1) / 2, kSplitRows / std::max<int64_t>(1, (int64_t)a.num_tokens * a.q_heads)}));
    };
    if (tile_box(p) == 0) return rows_kernel();
    if (a.shared_len > 0 && q_rows <= kTileKeys && (int64_t)a.num_tokens * a.q_heads <= kSplitRows) {
        // A prefix shared by short sequences: all their rows together against it, then each against its own keys.
        const int splits = splits_for((all_rows + kTileRows - 1) / kTileRows, a.shared_len);
        if (int rc = launch_tiles(p, a.head_dim, a.dtype, mods, true, splits, device, s)) return rc;
        p.prefix_splits = splits;
        p.shared_len = 0;
        return rows_kernel();
    }
    if (q_rows <= kRowTile) return rows_kernel();
    // Prompt chunks, and beside them (unless every sequence may be one) the sequences of few rows.
    const bool mixed = a.batch > 1 && a.num_tokens < (int64_t)a.batch * a.max_q_len;
    p.rows_limit = mixed ? kRowTile : 0;
    const int64_t row_tiles = std::max<int64_t>(1, all_rows / kTileRows);
    const int splits = splits_for(row_tiles, (int64_t)a.max_kv_len + a.shared_len);
    if (int rc = launch_tiles(p, a.head_dim, a.dtype, mods, false, splits, device, s)) return rc;
    return mixed ? rows_kernel() : KVX_OK;
}

}  // extern "C"
