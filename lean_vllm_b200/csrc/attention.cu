// Attention over the paged cache (kvx_attention).
//
// Mathematics. For a query row at position i, over the keys j that its mask leaves,
//     s_j = cap(scale q.k_j) + slope (j - i),   o = sum_j 2^(t_j - m) v_j / sum_j 2^(t_j - m),   t_j = s_j log2(e)
// in one pass with the running maximum m and sum of the softmax. Scores, maxima, sums and the accumulated output are
// held in 32 bits; the weights 2^(t_j - m) are rounded to the cache's 16-bit type for the tensor cores' second product:
// a relative rounding of at most 2^-8 in bf16 that averages out over the keys. They are at most 1 (attention_rows) or 2^8
// (attention_tiles, whose m may lag), far from the type's ends.

#include <algorithm>
#include <cmath>

#include "attention.cuh"

namespace {

using namespace kvx;

// ------------------------------------------------------------------------------------------------ rows kernel
//
// attention_rows: up to 8 or 16 query rows of one KV head (its group of query heads x the sequence's query tokens)
// against a stretch of a sequence's keys: the form for single tokens, bound by reading the cache.
//
// Work. The rows of a KV head share its keys, so a (sequence, KV head, tile of rows) group reads them once. Its keys are
// cut into tiles of 64 tokens; the tiles of all groups of all sequences, counted on the device from the lengths, are
// dealt out in equal contiguous runs to one wave of CTAs, whatever the lengths. A CTA's run covers whole groups and at
// most two partial ones; a partial group leaves (m, sum, o) in the workspace, and the CTA that brings the last part joins
// them in a fixed order (the result does not depend on which one that is).
//
// Inside a CTA each of the 4 warps takes its own 16 tokens of every tile with its own running maximum, sum and output,
// and loads them itself with cp.async into its own ring: no barrier until the group's end.
//
// Bound by HBM (graph-replayed times; calls take 0 to 3 us more): 64 ragged requests of up to 16k tokens (957 MB) take 156
// us, 6.1 TB/s; one of 131k 92 us, 5.8 TB/s: the walks end after 70 to 75 us on most SMs and 80 to 87 on the others, and 7
// are the join of 55 parts a head. 16 requests of 4 drafts over 8192 tokens (16 rows) take 96 us, 5.6 TB/s. One request of
// 317 tokens takes 7.2 us, a chain of waits: the launch, lengths, table, keys (0.5 us each) and the join of 5 parts.
//
// A window and a prefix mask leave keys between them that no row sees: the walk skips their tiles and fills what remains of
// them with zeros. A token with a window of 1024 and a prefix of 64 takes 9 us over 8k, 32k and 131k cached tokens alike.
//
// Up to 8 rows the products run transposed, S^T = K Q^T and O^T = V^T P^T, with the rows as the tensor cores' 8 columns:
// half the instructions and registers of a 16-row tile that would be half padding.

constexpr int kRowWarps = 4;
constexpr int kRowThreads = kRowWarps * 32;
constexpr int kWarpTokens = 16;
constexpr int kTileTokens = kRowWarps * kWarpTokens;

// Ring stages and CTAs per SM: 12 warps with 2 stages each or, where registers allow 8, with 3: 64 ragged requests take
// 162 us with 12 x 2 and 175 with 8 x 3, one of 131k tokens 98 and 96.
template <int ROWS>
struct RowShape {
    static constexpr int kStages = ROWS == 8 ? 2 : 3;
    static constexpr int kCtas = ROWS == 8 ? 3 : 2;
};

template <int D, int ROWS>
constexpr int kRowSmem = kRowWarps * RowShape<ROWS>::kStages * kWarpTokens * D * 2 * 2;

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

// The transpose of an 8 x 8 matrix of 16-bit elements, two of a row per lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// a / b for what nearly always fits 32 bits: a 64-bit division takes 400 cycles of a walk's 3000.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    if (((uint64_t)a | (uint64_t)b) >> 32 == 0) return (int64_t)((uint32_t)a / (uint32_t)b);
    return a / b;
}

// A sequence's share of the launch's tiles.
struct RowWork {
    int32_t lo;                // first key of the window, the prefix's lying ahead of it ...
    int32_t front, skip;       // ... in the first tiles of keys, behind which some are left out
    int32_t row_tiles, tiles;  // tiles of rows, tiles of keys per group
    __device__ __forceinline__ int64_t groups(const AttnParams &p) const { return (int64_t)row_tiles * p.kv_heads; }
};

template <int ROWS>
__device__ __forceinline__ RowWork row_work(const AttnParams &p, const Sequence &q) {
    RowWork w;
    w.lo = window_start(p, q.kv_len - q.q_len);
    w.front = (q.prefix + kTileTokens - 1) / kTileTokens;
    w.skip = max(0, w.lo / kTileTokens - w.front);
    w.row_tiles = (int32_t)(((int64_t)q.q_len * p.group + ROWS - 1) / ROWS);
    // An empty cache still gets one (empty) tile: its rows have to be written.
    w.tiles = max(1, (q.kv_len + kTileTokens - 1) / kTileTokens - w.skip);
    return w;
}

template <int ROWS>
__device__ __forceinline__ int64_t row_units(const AttnParams &p, int s) {
    if (blockIdx.x == 0 && (int64_t)p.kv_lens[s] > (int64_t)p.max_blocks * p.block_size)
        flag_error(p.error_word, p.status, kErrPastCache);
    const Sequence q = sequence_of(p, s);
    if ((int64_t)q.q_len * p.group > p.rows_limit) return 0;  // attention_tiles takes it
    const RowWork w = row_work<ROWS>(p, q);
    return w.groups(p) * w.tiles;
}

// Joins many parts of a group by way of shared memory, the ring's, half of it full of parts on their way while the other
// half is joined: registers hold 8 parts a thread, one wait for the L2 cache (1.1 us) after another, and 55 parts of 4 rows
// take 8 us so, 5 this way. (Up to 8 parts registers are as fast.)
template <int D, int ROWS, class FirstRow, class Finish>
__device__ __forceinline__ void join_many(const AttnParams &p, unsigned char *room, int parts, int rows,
                                          const FirstRow &first_row, const Finish &finish) {
    constexpr int kQuads = D / 4, kItems = ROWS * kQuads / kRowThreads, kHalf = kRowSmem<D, ROWS> / 2;
    static_assert(kHalf / (D * 4 + 8) <= kRowThreads, "a row of a part per thread");
    const int tid = threadIdx.x, values = rows * kQuads;  // float4 of a part
    const int at_once = kHalf / (rows * (D * 4 + 8));
    const int ml_part = tid / rows, ml_row = tid - ml_part * rows;  // the maximum and sum that this thread fetches
    Joined j[kItems];
    float2 ml_next = make_float2(0.f, 0.f);
    auto fetch = [&](int i0) {
        const int n = min(at_once, parts - i0);
        const uint32_t to = smem_u32(room) + (i0 / at_once & 1) * kHalf + tid * 16;
        if (ml_part < n) ml_next = __ldcg(&p.partial_ml[first_row(i0 + ml_part) + ml_row]);
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
            const float4 *from = reinterpret_cast<const float4 *>(p.partial_o) + first_row(i0 + i) * kQuads + tid;
#pragma unroll
            for (int k = 0; k < kItems; ++k)
                if (tid + k * kRowThreads < values)
                    cp_async16(to + i * values * 16 + k * kRowThreads * 16, from + k * kRowThreads, true);
        }
    };
    fetch(0);
    asm volatile("cp.async.commit_group;" ::: "memory");
    for (int i0 = 0; i0 < parts; i0 += at_once) {
        const int n = min(at_once, parts - i0);
        unsigned char *half = room + (i0 / at_once & 1) * kHalf;
        float2 *ml = reinterpret_cast<float2 *>(half + at_once * values * 16);  // [part][row]
        if (ml_part < n) ml[tid] = ml_next;
        if (i0 + at_once < parts) fetch(i0 + at_once);
        asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 1;" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            const int item = tid + k * kRowThreads, row = item / kQuads;
            if (item >= values) break;
            float top = j[k].top;
#pragma unroll 8
            for (int i = 0; i < n; ++i) top = fmaxf(top, ml[i * rows + row].x);
            const float reference = top == -INFINITY ? 0.f : top, own = exp2_fast(j[k].top - reference);
            j[k].top = top;
            j[k].sum *= own, j[k].o.x *= own, j[k].o.y *= own, j[k].o.z *= own, j[k].o.w *= own;
#pragma unroll 8
            for (int i = 0; i < n; ++i) {
                const float2 part = ml[i * rows + row];
                const float4 x = reinterpret_cast<const float4 *>(half)[i * values + item];
                const float f = exp2_fast(part.x - reference);
                j[k].sum += f * part.y;
                j[k].o.x += f * x.x, j[k].o.y += f * x.y, j[k].o.z += f * x.z, j[k].o.w += f * x.w;
            }
        }
        __syncthreads();  // this half is free again
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
        const int item = tid + k * kRowThreads;
        if (item < values) finish(item / kQuads, item % kQuads, j[k]);
    }
}

template <class T, int D, int ROWS, bool MODS>
__global__ void __launch_bounds__(kRowThreads, RowShape<ROWS>::kCtas)
attention_rows(const __grid_constant__ AttnParams p) {
    constexpr int kStages = RowShape<ROWS>::kStages;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int64_t scan[kRowWarps + 1];
    __shared__ int64_t found_start;
    __shared__ int found_sequence;
    __shared__ float2 warp_ml[kRowWarps][ROWS];
    __shared__ int is_last;

    launch_dependents();
    // Beside attention_tiles' part over a shared prefix nothing here waits for it: that kernel lets this one start after
    // its own wait, so everything before it is complete, and attention_join takes both parts.
    if (p.prefix_splits == 0) wait_prerequisites();

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    // ---- this CTA's run of tiles
    const int64_t own_units = tid < p.batch ? row_units<ROWS>(p, tid) : 0;  // of the first sequences, all there are often
    int64_t mine = own_units;
    for (int s = tid + kRowThreads; s < p.batch; s += kRowThreads) mine += row_units<ROWS>(p, s);
#pragma unroll
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(~0u, mine, o);
    if (lane == 0) scan[warp] = mine;
    __syncthreads();
    int64_t total = 0;
    for (int w = 0; w < kRowWarps; ++w) total += scan[w];
    const int64_t per_cta = max((int64_t)1, quotient(total + gridDim.x - 1, gridDim.x));
    int64_t unit = (int64_t)blockIdx.x * per_cta;
    const int64_t unit_end = min(total, unit + per_cta);
    if (unit >= unit_end) {
        wait_prerequisites();
        return;
    }
    int64_t before = 0;  // tiles of the sequences looked at so far
    for (int s0 = 0;; s0 += kRowThreads) {
        const int s = s0 + tid;
        const int64_t n = s0 == 0 ? own_units : s < p.batch ? row_units<ROWS>(p, s) : 0;
        int64_t sum = n;
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
    constexpr int kOutRow = D + 4;                    // floats of a row of a warp's output on its way to the join
    static_assert(ROWS * kOutRow * 4 <= kStages * 2 * kStageBytes, "a warp's output fits its ring");
    const uint32_t ring = smem_u32(smem) + warp * kStages * 2 * kStageBytes;
    float *my_o = reinterpret_cast<float *>(smem + warp * kStages * 2 * kStageBytes);  // once the ring is done with
    const float scale_log2 = p.scale * kLog2e;
    const float cap_in = p.softcap > 0.f ? scale_log2 * 2.f / p.softcap : 0.f, cap_out = p.softcap * kLog2e;
    // Blocks of whole stages: one lookup and one address a stage, the copies' a constant step apart.
    const bool stage_in_block = p.block_size % kWarpTokens == 0 && p.shared_len == 0;
    const int64_t copy_step = kPerCopy * p.token_stride;
    const uint32_t lane_to = (lane / kChunks) * D * 2;

    while (unit < unit_end) {
        const Sequence q = sequence_of(p, s);
        const RowWork work = row_work<ROWS>(p, q);
        const bool taken = (int64_t)q.q_len * p.group <= p.rows_limit;
        const int64_t s_end = taken ? s_start + work.groups(p) * work.tiles : s_start;
        if (unit >= s_end) {
            s_start = s_end;
            ++s;
            continue;
        }
        const int64_t in_sequence = unit - s_start;
        const int64_t group_index = quotient(in_sequence, work.tiles);
        const int tile0 = (int)(in_sequence - group_index * work.tiles);
        const int h = (int)(work.row_tiles == 1 ? group_index : quotient(group_index, work.row_tiles));
        const int row0 = (int)(group_index - (int64_t)h * work.row_tiles) * ROWS;
        const int64_t group_start = s_start + group_index * work.tiles, group_end = group_start + work.tiles;
        const int n_tiles = (int)(min(unit_end, group_end) - unit);
        const int rows = min(ROWS, q.q_len * p.group - row0);
        auto token_of = [&](int row) { return q.q_len == 1 ? 0 : (row0 + row) / p.group; };  // of the tile's rows
        auto head_of = [&](int row) { return h * p.group + row0 + row - token_of(row) * p.group; };
        auto query_of = [&](int row) -> uint64_t {
            if (row >= rows) return 0;
            return p.query + (int64_t)(q.q0 + token_of(row)) * p.q_token_stride + (int64_t)head_of(row) * p.q_head_stride;
        };
        // Stage i's first token, and which tokens are there: those from the window's first on, or (the modified form, which
        // calls with a window and a prefix take) all but those between the prefix and the window. One comparison instead of
        // two brings 64 ragged requests from 162 to 157 us.
        const int token0 = (tile0 + (MODS ? 0 : work.skip)) * kTileTokens + warp * kWarpTokens;
        auto stage_token = [&](int i) {
            return token0 + (i + (MODS && tile0 + i >= work.front ? work.skip : 0)) * kTileTokens;
        };
        const uint32_t gap = max(0, work.lo - q.prefix), span = max(0, q.kv_len - work.lo);
        auto readable = [&](int t) {
            return MODS ? t < q.kv_len && (uint32_t)(t - q.prefix) >= gap : (uint32_t)(t - work.lo) < span;
        };
        const int64_t lane_from = (int64_t)h * p.head_stride +
                                  (stage_in_block ? (lane / kChunks) * p.token_stride + (lane % kChunks) * 16 : 0);

        // Where stage i's tokens lie: in one block, this lane's first copy; else this lane's token (lanes 0-15). A byte
        // offset, or -1 where nothing is to be read.
        auto stage_offset = [&](int i) -> int64_t {
            if (i >= n_tiles) return -1;
            const int t = stage_token(i) + (stage_in_block ? 0 : lane);
            // (Of a stage in one block some token has to be there, so that the block's id is one.)
            if (stage_in_block ? t >= q.kv_len || (t + kWarpTokens <= work.lo && (!MODS || t >= q.prefix))
                               : lane >= kWarpTokens || !readable(t))
                return -1;
            const int64_t at = token_at(p, s, t);
            return at < 0 ? -1 : at + lane_from;
        };
        auto load_stage = [&](int i, int64_t offset) {
            const uint32_t k_stage = ring + (i % kStages) * 2 * kStageBytes + lane_to;
            if (stage_in_block) {
                const int t = stage_token(i) + lane / kChunks;
                uint64_t key = p.k_cache + (offset < 0 ? 0 : offset), value = p.v_cache + (offset < 0 ? 0 : offset);
#pragma unroll
                for (int c = 0; c < kCopies; ++c) {
                    const int token = c * kPerCopy + lane / kChunks;
                    const bool valid = offset >= 0 && readable(t + c * kPerCopy);
                    const uint32_t to = k_stage + c * kPerCopy * D * 2 + (((lane % kChunks) ^ (token & 7)) << 4);
                    cp_async16(to, reinterpret_cast<const void *>(key), valid);
                    cp_async16(to + kStageBytes, reinterpret_cast<const void *>(value), valid);
                    if (offset >= 0) key += copy_step, value += copy_step;
                }
            } else {
#pragma unroll
                for (int c = 0; c < kCopies; ++c) {
                    const int token = c * kPerCopy + lane / kChunks, chunk = lane % kChunks;
                    const int64_t at = __shfl_sync(~0u, offset, token);
                    const uint32_t to = k_stage + c * kPerCopy * D * 2 + ((chunk ^ (token & 7)) << 4);
                    const int64_t from = at < 0 ? 0 : at + chunk * 16;
                    cp_async16(to, reinterpret_cast<const void *>(p.k_cache + from), at >= 0);
                    cp_async16(to + kStageBytes, reinterpret_cast<const void *>(p.v_cache + from), at >= 0);
                }
            }
        };
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) {
            if (i < n_tiles) load_stage(i, stage_offset(i));
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        int64_t next_offset = stage_offset(kStages - 1);

        // ---- queries, in the registers of the first product, and what this lane's two rows see
        constexpr int kQueryRegs = ROWS == 8 ? 2 : 4;
        uint32_t qf[D / 16][kQueryRegs];
        if (ROWS == 8) {  // row lane / 4 as a column
            const int row = lane / 4;
            const uint64_t at = query_of(row);
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    qf[k][half] = at ? *reinterpret_cast<const uint32_t *>(at + (k * 16 + half * 8 + (lane & 3) * 2) * 2) : 0u;
        } else {  // rows lane / 4 and lane / 4 + 8
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = lane / 4 + 8 * r;
                const uint64_t at = query_of(row);
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
#pragma unroll
                    for (int half = 0; half < 2; ++half)
                        qf[k][(r + 2 * half) % kQueryRegs] =
                            at ? *reinterpret_cast<const uint32_t *>(at + (k * 16 + half * 8 + (lane & 3) * 2) * 2) : 0u;
            }
        }
        int position[2], prefix[2];  // of rows 2 (lane % 4) + r, or lane / 4 + 8 r
        float slope[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = ROWS == 8 ? 2 * (lane & 3) + r : lane / 4 + 8 * r;
            const bool valid = row < rows;
            position[r] = valid ? q.kv_len - q.q_len + token_of(row) : -1;
            prefix[r] = valid ? q.prefix : 0;
            slope[r] = MODS && valid && p.slopes ? p.slopes[head_of(row)] * kLog2e : 0.f;
        }
        // Every row of the tile sees the keys from see_lo up to see_hi: whole stages in there need no mask.
        const int first_position = q.kv_len - q.q_len + token_of(0);
        const int last_position = q.kv_len - q.q_len + token_of(rows - 1);
        const int see_lo = window_start(p, last_position);
        const int see_hi = min(q.kv_len, first_position + 1);

        // ---- the walk over the keys. c holds a stage's 16 tokens x ROWS scores: c[n][e] belongs to this lane's row
        // e / 2 (16 rows: token 8 n + 2 (lane % 4) + e % 2) or e % 2 (8 rows: token lane / 4 + 8 (e / 2)).
        constexpr int kScores = ROWS == 8 ? 1 : 2, kOut = ROWS == 8 ? D / 16 : D / 8;
        float m[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f}, o[kOut][4];
#pragma unroll
        for (int n = 0; n < kOut; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;

        for (int i = 0; i < n_tiles; ++i) {
            if (i + kStages - 1 < n_tiles) load_stage(i + kStages - 1, next_offset);
            asm volatile("cp.async.commit_group;" ::: "memory");
            next_offset = stage_offset(i + kStages);
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
            __syncwarp();
            const uint32_t k_stage = ring + (i % kStages) * 2 * kStageBytes, v_stage = k_stage + kStageBytes;
            const int t0 = stage_token(i);

            float c[kScores][4] = {};
            if (ROWS == 8) {
                float odd[4] = {};
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    uint32_t a[4];
                    const int token = lane & 15, chunk = 2 * k + (lane >> 4);
                    ldmatrix4(a, k_stage + token * D * 2 + ((chunk ^ (token & 7)) << 4));
                    mma16816<T>(k & 1 ? odd : c[0], a, qf[k][0], qf[k][1]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) c[0][e] += odd[e];
            } else {
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    uint32_t b[4];
                    const int token = (lane & 7) + ((lane & 16) >> 1), chunk = 2 * k + ((lane >> 3) & 1);
                    ldmatrix4(b, k_stage + token * D * 2 + ((chunk ^ (token & 7)) << 4));
                    mma16816<T>(c[0], qf[k], b[0], b[1]);
                    mma16816<T>(c[kScores - 1], qf[k], b[2], b[3]);
                }
            }
            const bool masked = t0 < see_lo || t0 + kWarpTokens > see_hi;
            float stage_max[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < kScores; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = ROWS == 8 ? e & 1 : e >> 1;
                    const int t = t0 + (ROWS == 8 ? lane / 4 + 8 * (e >> 1) : n * 8 + (lane & 3) * 2 + (e & 1));
                    float x;  // the score times log2(e)
                    if (MODS) {
                        // tanh(z) = 1 - 2 / (e^2z + 1), to 2^-22 of the cap, where the exponent's error counts
                        x = p.softcap > 0.f ? cap_out - 2.f * cap_out * reciprocal_fast(exp2_fast(c[n][e] * cap_in) + 1.f)
                                            : c[n][e] * scale_log2;
                        x += slope[r] * (float)(t - position[r]);
                    } else {
                        x = c[n][e] * scale_log2;
                    }
                    if (masked) {
                        const bool seen = t < q.kv_len &&
                                          ((t <= position[r] && (p.window <= 0 || t > position[r] - p.window)) ||
                                           t < prefix[r]);
                        x = seen ? x : -INFINITY;
                    }
                    c[n][e] = x;
                    stage_max[r] = fmaxf(stage_max[r], x);
                }
            bool grown = false;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                if (ROWS == 8) {
                    stage_max[r] = fmaxf(stage_max[r], __shfl_xor_sync(~0u, stage_max[r], 4));
                    stage_max[r] = fmaxf(stage_max[r], __shfl_xor_sync(~0u, stage_max[r], 8));
                    stage_max[r] = fmaxf(stage_max[r], __shfl_xor_sync(~0u, stage_max[r], 16));
                } else {
                    stage_max[r] = fmaxf(stage_max[r], __shfl_xor_sync(~0u, stage_max[r], 1));
                    stage_max[r] = fmaxf(stage_max[r], __shfl_xor_sync(~0u, stage_max[r], 2));
                }
                grown |= stage_max[r] > m[r];
            }
            if (__any_sync(~0u, grown)) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float now = fmaxf(m[r], stage_max[r]), factor = weight_of(m[r], now);
                    m[r] = now;
                    sum[r] *= factor;
#pragma unroll
                    for (int n = 0; n < kOut; ++n) {
                        o[n][ROWS == 8 ? r : 2 * r] *= factor;
                        o[n][ROWS == 8 ? r + 2 : 2 * r + 1] *= factor;
                    }
                }
            }
            const float reference[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
            for (int n = 0; n < kScores; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = ROWS == 8 ? e & 1 : e >> 1;
                    c[n][e] = exp2_fast(c[n][e] - reference[r]);
                    sum[r] += c[n][e];
                }
            if (ROWS == 8) {
                // Weights by (token, row) pairs become the second product's (row, token) ones.
                const uint32_t b0 = transpose8(Pack2<T>::of(c[0][0], c[0][1]));
                const uint32_t b1 = transpose8(Pack2<T>::of(c[0][2], c[0][3]));
#pragma unroll
                for (int n = 0; n < D / 16; ++n) {
                    uint32_t a[4];
                    const int token = (lane & 7) + ((lane & 16) >> 1), chunk = 2 * n + ((lane >> 3) & 1);
                    ldmatrix4_trans(a, v_stage + token * D * 2 + ((chunk ^ (token & 7)) << 4));
                    mma16816<T>(o[n], a, b0, b1);
                }
            } else {
                constexpr int kLast = kScores - 1;
                const uint32_t pa[4] = {Pack2<T>::of(c[0][0], c[0][1]), Pack2<T>::of(c[0][2], c[0][3]),
                                        Pack2<T>::of(c[kLast][0], c[kLast][1]), Pack2<T>::of(c[kLast][2], c[kLast][3])};
#pragma unroll
                for (int n = 0; n < D / 8; n += 2) {
                    uint32_t b[4];
                    const int token = lane & 15, chunk = n + (lane >> 4);
                    ldmatrix4_trans(b, v_stage + token * D * 2 + ((chunk ^ (token & 7)) << 4));
                    mma16816<T>(o[n % kOut], pa, b[0], b[1]);
                    mma16816<T>(o[(n + 1) % kOut], pa, b[2], b[3]);
                }
            }
            __syncwarp();
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();

        // ---- join the warps
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if (ROWS == 8) {
                sum[r] += __shfl_xor_sync(~0u, sum[r], 4);
                sum[r] += __shfl_xor_sync(~0u, sum[r], 8);
                sum[r] += __shfl_xor_sync(~0u, sum[r], 16);
                const int row = 2 * (lane & 3) + r;
                if (lane < 4) warp_ml[warp][row] = make_float2(m[r], sum[r]);
#pragma unroll
                for (int n = 0; n < kOut; ++n) {
                    my_o[row * kOutRow + n * 16 + lane / 4] = o[n][r];
                    my_o[row * kOutRow + n * 16 + lane / 4 + 8] = o[n][r + 2];
                }
            } else {
                sum[r] += __shfl_xor_sync(~0u, sum[r], 1);
                sum[r] += __shfl_xor_sync(~0u, sum[r], 2);
                const int row = (lane / 4 + 8 * r) % ROWS;
                if ((lane & 3) == 0) warp_ml[warp][row] = make_float2(m[r], sum[r]);
#pragma unroll
                for (int n = 0; n < kOut; ++n)
                    *reinterpret_cast<float2 *>(my_o + row * kOutRow + n * 8 + (lane & 3) * 2) =
                        make_float2(o[n][2 * r], o[n][2 * r + 1]);
            }
        }
        __syncthreads();
        const bool whole = unit == group_start && n_tiles == work.tiles;
        const int slot = 2 * blockIdx.x + (unit == group_start ? 1 : 0);
        constexpr int kQuads = D / 4;
        constexpr int kWarpFloats = kStages * 2 * kStageBytes / 4;
        const float *all_o = reinterpret_cast<const float *>(smem);

        // A row's four elements, done but for a shared prefix: into the output, or as one more part for attention_join.
        auto finish = [&](int row, int quad, const Joined &j) {
            const int token = q.q0 + token_of(row), head = head_of(row);
            if (p.prefix_splits > 0) {
                const int64_t at = ((int64_t)p.prefix_splits * p.num_tokens + token) * p.q_heads + head;
                reinterpret_cast<float4 *>(p.split_o)[at * kQuads + quad] = j.o;
                if (quad == 0) p.split_ml[at] = make_float2(j.top, j.sum);
            } else {
                write_row<T>(p, token, head, quad, j);
            }
        };
        for (int item = tid; item < rows * kQuads; item += kRowThreads) {
            const int row = item / kQuads, quad = item % kQuads;
            Joined j;
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) j.top = fmaxf(j.top, warp_ml[w][row].x);
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) {
                const float f = weight_of(warp_ml[w][row].x, j.top);
                const float4 x = reinterpret_cast<const float4 *>(all_o + w * kWarpFloats + row * kOutRow)[quad];
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
            const int c0 = (int)quotient(group_start, per_cta), c1 = (int)quotient(group_end - 1, per_cta);
            __syncthreads();
            if (tid == 0) {
                __threadfence();  // orders what the barrier made this thread's to know, the other threads' writes
                is_last = atomicAdd(&p.counters[c0], 1) == c1 - c0;
                if (is_last) p.counters[c0] = 0;  // for the next launch
            }
            __syncthreads();
            if (is_last) {
                __threadfence();
                const int parts = c1 - c0 + 1;
                auto first_row = [&](int i) { return (int64_t)(2 * (c0 + i) + (i == 0)) * kRowTile; };  // of part i
                if (parts <= 8) {
                    for (int item = tid; item < rows * kQuads; item += kRowThreads) {
                        const int row = item / kQuads, quad = item % kQuads;
                        Joined j;
                        join_parts(j, parts, p.partial_ml, p.partial_o, kQuads, quad,
                                   [&](int i) { return first_row(i) + row; });
                        finish(row, quad, j);
                    }
                } else {
                    join_many<D, ROWS>(p, smem, parts, rows, first_row, finish);
                }
            }
        }
        __syncthreads();  // the ring and the joined values are free again
        unit += n_tiles;
    }
    wait_prerequisites();
}

// Joins each row's parts: attention_tiles' splits, or its splits of a shared prefix and attention_rows' part over the
// sequence's own keys. Rows of sequences that attention_rows took whole have none.
//
// A thread has four elements of a row, and at_once parts of them on their way into its own places in shared memory at a
// time; the threads of a row fetch the parts' maxima and sums, up to two each. Bound by the L2 cache's latency, so
// everything is asked for at once: 64 requests of 32 heads behind 8192 tokens (2048 rows of 19 parts) take 36 us, 40 with
// 8 parts at a time in registers; 500 of them (5 parts) 133 and 135.
constexpr int kJoinThreads = 128;
template <int D>
constexpr int kJoinAtOnce = D == 128 ? 48 : 32;  // two for each of a row's threads, 96 KB of shared memory at most

template <class T, int D>
__global__ void __launch_bounds__(kJoinThreads)
attention_join(const __grid_constant__ AttnParams p, int parts, int at_once, bool mixed) {
    constexpr uint32_t kQuads = D / 4, kRows = kJoinThreads / kQuads;
    extern __shared__ __align__(128) unsigned char smem[];  // [part][thread]
    const uint32_t rows = (uint32_t)p.num_tokens * p.q_heads;  // at most kSplitRows
    const uint32_t quad = threadIdx.x % kQuads, row = blockIdx.x * kRows + threadIdx.x / kQuads;
    const int token = (int)(row / (uint32_t)p.q_heads);
    wait_prerequisites();
    launch_dependents();
    if (row >= rows) return;
    if (mixed && (int64_t)sequence_of(p, sequence_at(p, token)).q_len * p.group <= p.rows_limit) return;
    const uint32_t mask = kQuads == 32 ? ~0u : 0xffffu << (threadIdx.x & 16);  // the row's threads
    const float4 *mine = reinterpret_cast<const float4 *>(smem) + threadIdx.x;
    Joined j;
    for (int i0 = 0; i0 < parts; i0 += at_once) {
        const int n = min(at_once, parts - i0);
        float2 ml[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int i = quad + k * kQuads;
            ml[k] = i < n ? __ldcg(&p.split_ml[row + (int64_t)(i0 + i) * rows]) : make_float2(-INFINITY, 0.f);
        }
        const float4 *from = reinterpret_cast<const float4 *>(p.split_o) + (row + (int64_t)i0 * rows) * kQuads + quad;
        for (int i = 0; i < n; ++i, from += (int64_t)rows * kQuads)
            cp_async16(smem_u32(mine + i * kJoinThreads), from, true);
        asm volatile("cp.async.commit_group;" ::: "memory");
        float top = fmaxf(j.top, fmaxf(ml[0].x, ml[1].x));
#pragma unroll
        for (int o = kQuads / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(mask, top, o));
        const float reference = top == -INFINITY ? 0.f : top, own = exp2_fast(j.top - reference);
        const float f[2] = {exp2_fast(ml[0].x - reference), exp2_fast(ml[1].x - reference)};
        float sum = f[0] * ml[0].y + f[1] * ml[1].y;
#pragma unroll
        for (int o = kQuads / 2; o; o >>= 1) sum += __shfl_xor_sync(mask, sum, o);
        j.top = top;
        j.sum = j.sum * own + sum;
        j.o.x *= own, j.o.y *= own, j.o.z *= own, j.o.w *= own;
        asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
            const float factor = __shfl_sync(mask, i < (int)kQuads ? f[0] : f[1], i % kQuads, kQuads);
            const float4 x = mine[i * kJoinThreads];
            j.o.x += factor * x.x, j.o.y += factor * x.y, j.o.z += factor * x.z, j.o.w += factor * x.w;
        }
    }
    write_row<T>(p, token, (int)(row - token * p.q_heads), quad, j);
}

// ------------------------------------------------------------------------------------------------ host side

constexpr size_t kRowPartials = (size_t)kMaxRowCtas * 2 * kRowTile;
constexpr size_t kMlBytes = sizeof(float2), kOutBytes = 128 * sizeof(float);
constexpr size_t kSplitAt = KVX_ATTENTION_ZEROED + kRowPartials * (kMlBytes + kOutBytes);
constexpr size_t kWorkspaceBytes = kSplitAt + kSplitRows * (kMlBytes + kOutBytes);
static_assert(kMaxRowCtas <= kTileCounter && (kTileCounter + 1) * sizeof(int32_t) <= KVX_ATTENTION_ZEROED, "counters");

template <class T, int D, int ROWS, bool MODS>
int launch_rows(const AttnParams &p, const Device &device, const Queue &queue) {
    static AllowedSmem allowed;
    auto kernel = attention_rows<T, D, ROWS, MODS>;
    if (int rc = allowed.allow(kernel, kRowSmem<D, ROWS>, device.index)) return rc;
    return launch(kernel, std::min(RowShape<ROWS>::kCtas * device.sms, kMaxRowCtas), kRowThreads, kRowSmem<D, ROWS>,
                  queue, p);
}

template <class T, int D>
int launch_rows(const AttnParams &p, int rows, bool mods, const Device &device, const Queue &queue) {
    if (rows <= 8) return mods ? launch_rows<T, D, 8, true>(p, device, queue) : launch_rows<T, D, 8, false>(p, device, queue);
    return mods ? launch_rows<T, D, 16, true>(p, device, queue) : launch_rows<T, D, 16, false>(p, device, queue);
}

template <class T, int D>
int launch_join(const AttnParams &p, int parts, bool mixed, const Device &device, const Queue &queue) {
    const int64_t rows = (int64_t)p.num_tokens * p.q_heads;
    constexpr int kRows = 4 * kJoinThreads / D, kAtOnce = kJoinAtOnce<D>;
    const int rounds = (parts + kAtOnce - 1) / kAtOnce, at_once = (parts + rounds - 1) / rounds;
    static AllowedSmem allowed;
    auto kernel = attention_join<T, D>;
    if (int rc = allowed.allow(kernel, kAtOnce * kJoinThreads * 16, device.index)) return rc;
    return launch(kernel, (rows + kRows - 1) / kRows, kJoinThreads, at_once * kJoinThreads * 16, queue, p,
                  parts, at_once, mixed);
}

// How many parts attention_tiles' items are cut into along the keys: more items fill SMs that would idle, but every part
// of a row is written and read once more. By what both take on B200 (us): a pair of tiles 1.85, an item's ends 1.2, the
// join 3 and its traffic at 4 TB/s. 200 tokens of 32 heads behind 4k take 60 us in one part, 29 in four; 512 new tokens
// 14 in one, 18 in two.
int choose_splits(int64_t items, int64_t keys, int64_t rows, int head_dim, int ctas) {
    const int64_t tiles = std::max<int64_t>(1, (keys + kTileKeys - 1) / kTileKeys);
    const double part_bytes = 2.0 * rows * (4 * head_dim + 8);
    int best = 1;
    double least = 0;
    for (int splits = 1; splits <= ctas && splits * rows <= kSplitRows && (splits == 1 || 2 * splits <= tiles + 1); ++splits) {
        const double rounds = (double)((items * splits + ctas - 1) / ctas);
        double us = rounds * (1.85 * (double)((tiles + splits - 1) / splits) + 1.2);
        if (splits > 1) us += 3 + splits * part_bytes / 4e6;
        if (splits == 1 || us < least) best = splits, least = us;
    }
    return best;
}

}  // namespace

extern "C" {

uint64_t kvx_attention_workspace_bytes(void) { return kWorkspaceBytes; }

int kvx_attention(const kvx_attention_args *args, int flags, void *stream) {
    Range range("kvx_attention");
    if (!args) return fail(KVX_ERR_INVALID, "null arguments");
    if (flags & ~KVX_STORE_SERIAL) return fail(KVX_ERR_INVALID, "flags %#x; KVX_STORE_SERIAL is the one there is", flags);
    const kvx_attention_args &a = *args;
    if (a.num_tokens < 0 || a.batch < 0) return fail(KVX_ERR_INVALID, "%d tokens of %d sequences", a.num_tokens, a.batch);
    if (a.q_heads < 1 || a.kv_heads < 1 || a.q_heads % a.kv_heads != 0)
        return fail(KVX_ERR_INVALID, "%d query heads over %d KV heads", a.q_heads, a.kv_heads);
    if (a.head_dim != 64 && a.head_dim != 128) return fail(KVX_ERR_INVALID, "head_dim %d; 64 or 128", a.head_dim);
    if (a.dtype != KVX_BF16 && a.dtype != KVX_FP16) return fail(KVX_ERR_INVALID, "unknown element type %d", a.dtype);
    if (a.block_size < 1 || a.num_blocks < 0 || a.max_blocks < 0 || a.table_stride < 0 || a.shared_len < 0 ||
        a.shared_blocks < 0)
        return fail(KVX_ERR_INVALID, "bad block size, block count or table");
    // Positions and the ends of tiles stay below 2^31.
    if ((int64_t)a.max_blocks * a.block_size + a.shared_len > ((int64_t)1 << 31) - 1024)
        return fail(KVX_ERR_INVALID, "more than 2^31 - 1024 tokens a sequence");
    if (a.window < 0 || !(a.softcap >= 0.f)) return fail(KVX_ERR_INVALID, "negative window or softcap");
    if (std::isinf(a.softcap)) return fail(KVX_ERR_INVALID, "an infinite softcap; 0 is none");
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
    const Queue queue{static_cast<cudaStream_t>(stream), (flags & KVX_STORE_SERIAL) != 0};
    // Without q_starts every sequence has one query token, whatever bound came with the call.
    const int64_t max_q_len = a.q_starts ? std::max(a.max_q_len, 1) : 1;
    const int64_t q_rows = max_q_len * p.group;  // of the longest sequence and one KV head
    const bool row_mods = mods || (a.window > 0 && a.prefix_lens);
    auto rows_kernel = [&](int64_t rows) {
        const int n = rows <= 8 ? 8 : 16;
        if (a.head_dim == 128)
            return a.dtype == KVX_BF16 ? launch_rows<__nv_bfloat16, 128>(p, n, row_mods, device, queue)
                                       : launch_rows<__half, 128>(p, n, row_mods, device, queue);
        return a.dtype == KVX_BF16 ? launch_rows<__nv_bfloat16, 64>(p, n, row_mods, device, queue)
                                   : launch_rows<__half, 64>(p, n, row_mods, device, queue);
    };

    auto join = [&](int parts, bool mixed) {
        if (a.head_dim == 128)
            return a.dtype == KVX_BF16 ? launch_join<__nv_bfloat16, 128>(p, parts, mixed, device, queue)
                                       : launch_join<__half, 128>(p, parts, mixed, device, queue);
        return a.dtype == KVX_BF16 ? launch_join<__nv_bfloat16, 64>(p, parts, mixed, device, queue)
                                   : launch_join<__half, 64>(p, parts, mixed, device, queue);
    };

    // ---- which kernel takes what
    if (tile_box(p) == 0) return rows_kernel(q_rows);
    const int64_t rows = (int64_t)a.num_tokens * a.q_heads;
    const int64_t tile_tokens = 128 / p.group;
    if (a.shared_len > 0 && q_rows <= kTileKeys && 2 * p.q_heads <= kSplitRows) {
        // A prefix shared by short sequences: all their rows together against it, each against its own keys, both joined.
        // One item per CTA: its parts are a part more of every row either way. Items of one tile of rows: 64 requests
        // behind 8192 tokens take 35.9 us, 36.3 with two tiles (64-wide heads: 27.6 and 28.8). A batch whose parts pass the
        // workspace goes in equal runs of tokens, the prefix read once for each.
        const int64_t runs = (2 * rows + kSplitRows - 1) / kSplitRows;
        const int run_tokens = (int)((a.num_tokens + runs - 1) / runs);
        for (int token0 = 0; token0 < a.num_tokens; token0 += run_tokens) {
            p.token0 = token0;
            p.num_tokens = std::min(run_tokens, a.num_tokens - token0);
            p.query = (uint64_t)(uintptr_t)a.query + token0 * a.q_token_stride;
            p.out = (uint64_t)(uintptr_t)a.out + token0 * a.out_token_stride;
            const int64_t items = (p.num_tokens + tile_tokens - 1) / tile_tokens * p.kv_heads;
            const int64_t tiles = (a.shared_len + kTileKeys - 1) / kTileKeys;
            const int64_t most = kSplitRows / ((int64_t)p.num_tokens * a.q_heads) - 1;
            const int splits = (int)std::max<int64_t>(1, std::min({2 * device.sms / items, (tiles + 1) / 2, most}));
            p.prefix_splits = 0;
            p.shared_len = a.shared_len;
            if (int rc = launch_tiles(p, a.head_dim, a.dtype, mods, true, 1, splits, device, queue)) return rc;
            p.prefix_splits = splits;
            p.shared_len = 0;
            if (int rc = rows_kernel(q_rows)) return rc;
            if (int rc = join(splits + 1, false)) return rc;
        }
        return KVX_OK;
    }
    if (q_rows <= kRowTile) return rows_kernel(q_rows);
    // Prompt chunks, and beside them (unless every sequence may be one) the sequences of few rows.
    const bool mixed = a.batch > 1 && a.num_tokens < a.batch * max_q_len;
    p.rows_limit = !mixed ? 0 : p.group <= 8 ? 8 : kRowTile;
    auto items_of = [&](int groups) {  // about how many
        const int64_t tokens = groups * tile_tokens;
        int64_t items = a.batch * ((max_q_len + tokens - 1) / tokens);
        if (mixed) items = std::min<int64_t>(items, (a.num_tokens + tokens - 1) / tokens + (a.batch - 1) / 2);
        return std::max<int64_t>(1, items) * p.kv_heads;
    };
    auto splits_of = [&](int groups) {
        int64_t keys = (int64_t)a.max_kv_len + a.shared_len;
        if (a.window > 0 && !a.prefix_lens) keys = std::min<int64_t>(keys, a.window + groups * tile_tokens);
        return choose_splits(items_of(groups), keys, rows, a.head_dim, device.sms * (3 - groups));
    };
    // Two tiles of rows on one CTA per SM bring the same keys for both; one tile on each of two CTAs lets a few items
    // spread over more SMs, and the two fall less into step. 128 wide, 32 heads over 8: a prompt of 512 tokens (64 pairs
    // for 148 SMs) takes 15.8 us in pairs and 14.3 in single tiles, 768 tokens 19.7 and 19.3, 1024 24.1 and 24.6, 2048
    // 53.2 and 57.0. 64 wide, the single tile is ahead at every size: 13.4 and 11.1, 45.4 and 42.1, 8192 tokens 418 and 389.
    int groups = 1, splits = 0;
    if (a.head_dim == 128 && max_q_len > tile_tokens) {
        splits = splits_of(2);
        if (items_of(2) * splits * 8 > (int64_t)device.sms * 5) groups = 2;
    }
    if (groups == 1) splits = splits_of(1);
    if (int rc = launch_tiles(p, a.head_dim, a.dtype, mods, false, groups, splits, device, queue)) return rc;
    if (splits > 1)
        if (int rc = join(splits, mixed)) return rc;
    return mixed ? rows_kernel(p.rows_limit) : KVX_OK;
}

}  // extern "C"
