// attention_tiles: up to 256 query rows of one KV head against a stretch of keys, on the 5th-generation tensor cores:
// the form for prompts, drafted tokens in numbers, and a prefix that a whole batch shares, where a key meets so many
// rows that the products bound the time, not the cache.
//
// Work. The query rows of a KV head (its group of heads x the sequence's query tokens, or the whole batch's for a shared
// prefix) share its keys. A CTA takes 256 of them, as two tiles of 128, and walks its keys in tiles of 128. For each
// pair of tiles, S = Q K^T and O += P V are one chain of tcgen05.mma each, 128 x 128 x D and 128 x D x 128, with Q, K and
// V in shared memory and S, P and O in TMEM (S, then P in its place, 128 columns a tile; O, D columns a tile).
//
// Roles. One warp copies K and V tiles by TMA into a ring; one thread issues the products; two groups of 4 warps run the
// softmax of a tile each, one row per thread. While one tile's scores are in the softmax the other's products run.
//
// The running maximum moves only when a tile's exceeds it by more than 2^8 (kLazy): the weights then stay below 2^8, which
// costs no precision in a floating type, and the accumulated output is rescaled a few times per row, not per tile.

#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "attention.cuh"

namespace {

using namespace kvx;

constexpr int kSoftmaxWarps = 8;
constexpr int kIssueWarp = 8;
constexpr int kLoadWarp = 9;
constexpr int kThreads = 384;
// The launch gives each thread 168 registers; a row's 128 scores want more, the other warps less:
// 256 x 224 + 128 x 56 = 64512, the launch's 384 x 168.
constexpr int kSoftmaxRegisters = 224, kOtherRegisters = 56;
constexpr float kLazy = 8.f;
constexpr uint64_t kWaitNs = 2000000000ull;  // a wait that has not ended after 2 s is an error

template <int D>
struct Shape {
    static constexpr int kHalves = D / 64;                      // 128-byte columns of a row
    static constexpr int kTileBytes = kTileKeys * D * 2;        // of 128 rows: queries, keys or values
    static constexpr int kHalfBytes = kTileKeys * 128;
    static constexpr int kSlots = D == 128 ? 5 : 10;            // ring of K and V tiles: 160 KB
    static constexpr int kBytes = (2 + kSlots) * kTileBytes + 1024;
    static constexpr int kOutColumn = 256;                      // TMEM: S and P of both tiles, then O of both
};

struct TileParams {
    AttnParams a;
    CUtensorMap keys, values;
    int32_t box;          // tokens per copy
    int32_t splits;
    int32_t prefix_only;
    int32_t row_tiles;    // bound on the launch's tiles of 256 rows
};

struct Item {
    Sequence q;
    int32_t sequence, head, row0, rows, split;
    int32_t lo, hi;              // own keys that any row sees
    int32_t shared_tiles, tiles; // tiles of the shared prefix walked first, and all of this split's ...
    int32_t first_tile;          // ... from this one of the item's on
    int32_t lo_tile;             // first tile of own keys
};

// ---- tcgen05

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// A shared-memory operand: rows (or columns) of 128 bytes, swizzled in groups of 8 (1024 bytes).
// `leading`: bytes between the 64-element halves of an operand whose contiguous direction is not the summed one.
__device__ __forceinline__ uint64_t operand(uint32_t address, uint32_t leading) {
    return (uint64_t)((address & 0x3ffff) >> 4) | (uint64_t)(leading >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

template <class T>
__host__ __device__ constexpr uint32_t instruction(int n, bool b_transposed) {
    constexpr uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    return 1u << 4 | type << 7 | type << 10 | (b_transposed ? 1u : 0u) << 16 | (uint32_t)(n >> 3) << 17 |
           (uint32_t)(128 >> 4) << 24;
}

__device__ __forceinline__ void mma_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t inst, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(inst), "r"((uint32_t)accumulate)
        : "memory");
}

__device__ __forceinline__ void mma_tensor(uint32_t d, uint32_t a, uint64_t b, uint32_t inst, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(inst), "r"((uint32_t)accumulate)
        : "memory");
}

__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

// Arrives on `bar` once every product issued so far has completed.
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void load32(uint32_t address, float (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
          "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
          "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
          "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(address));
}

__device__ __forceinline__ void load16(uint32_t address, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(address));
}

__device__ __forceinline__ void store32(uint32_t address, const float (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(address),
        "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]), "f"(r[8]), "f"(r[9]),
        "f"(r[10]), "f"(r[11]), "f"(r[12]), "f"(r[13]), "f"(r[14]), "f"(r[15]), "f"(r[16]), "f"(r[17]), "f"(r[18]),
        "f"(r[19]), "f"(r[20]), "f"(r[21]), "f"(r[22]), "f"(r[23]), "f"(r[24]), "f"(r[25]), "f"(r[26]), "f"(r[27]),
        "f"(r[28]), "f"(r[29]), "f"(r[30]), "f"(r[31])
        : "memory");
}

__device__ __forceinline__ void store16(uint32_t address, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(address),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap *map, int x, int token, int head, int block,
                                         uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(token), "r"(head), "r"(block), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
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

__device__ __forceinline__ float max_of(float top, const float (&x)[32]) {
    float a = top, b = x[0];
#pragma unroll
    for (int e = 1; e + 3 < 32; e += 4) {
        asm("max.f32 %0, %0, %1, %2;" : "+f"(a) : "f"(x[e]), "f"(x[e + 1]));
        asm("max.f32 %0, %0, %1, %2;" : "+f"(b) : "f"(x[e + 2]), "f"(x[e + 3]));
    }
    asm("max.f32 %0, %0, %1, %2;" : "+f"(a) : "f"(x[29]), "f"(x[30]));
    return fmaxf(fmaxf(a, b), x[31]);
}

// Waits for a phase of `bar`, for as long as no wait of the CTA has run out.
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity, volatile int *gave_up) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t deadline = globaltimer() + kWaitNs;
    while (!mbar_try_wait(bar, parity)) {
        if (*gave_up) return false;
        if (globaltimer() > deadline) {
            *gave_up = 1;
            return false;
        }
    }
    return true;
}

// The same for a whole warp, which stays together whether the wait ends or runs out.
__device__ __forceinline__ bool warp_waits(uint32_t bar, uint32_t parity, volatile int *gave_up) {
    return __all_sync(~0u, wait_phase(bar, parity, gave_up));
}

// The CTA's item: which rows of which sequence, and which keys. Row tiles come last first, since the last ones of a
// causal prompt see the most keys. Every thread of warp 0 calls this; false: no work.
__device__ bool find_item(const TileParams &t, int id, Item &item) {
    const AttnParams &p = t.a;
    const int lane = threadIdx.x & 31;
    const int per_tile = p.kv_heads * t.splits;
    const int r = id / per_tile;
    item.split = (id - r * per_tile) / p.kv_heads;
    item.head = id - r * per_tile - item.split * p.kv_heads;
    if (t.prefix_only) {
        item.sequence = 0;
        item.q = Sequence{0, p.num_tokens, p.shared_len, 0};
        item.row0 = r * kTileRows;
        item.rows = min(kTileRows, p.num_tokens * p.group - item.row0);
        item.lo = item.hi = item.lo_tile = 0;
        item.shared_tiles = (p.shared_len + kTileKeys - 1) / kTileKeys;
        item.tiles = item.shared_tiles;
    } else {
        auto tiles_of = [&](const Sequence &q) {
            const int64_t rows = (int64_t)q.q_len * p.group;
            return rows > p.rows_limit ? (int)((rows + kTileRows - 1) / kTileRows) : 0;
        };
        auto at = [&](int s) { return s < p.batch ? sequence_of(p, s) : Sequence{0, 0, 0, 0}; };
        Sequence mine = at(lane);  // of the 32 sequences looked at now: all there are, often
        int n = tiles_of(mine), total = n;
        for (int s = lane + 32; s < p.batch; s += 32) total += tiles_of(at(s));
        total = __reduce_add_sync(~0u, total);
        const int wanted = total - 1 - r;
        if (wanted < 0) return false;
        int before = 0;
        for (int s0 = 0;;) {
            int sum = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(~0u, sum, o);
                if (lane >= o) sum += up;
            }
            const unsigned here = __ballot_sync(~0u, before + sum > wanted);
            if (here) {
                const int who = __ffs(here) - 1;
                item.sequence = s0 + who;
                item.row0 = (wanted - before - __shfl_sync(~0u, sum - n, who)) * kTileRows;
                item.q = Sequence{__shfl_sync(~0u, mine.q0, who), __shfl_sync(~0u, mine.q_len, who),
                                  __shfl_sync(~0u, mine.kv_len, who), __shfl_sync(~0u, mine.prefix, who)};
                break;
            }
            before += __shfl_sync(~0u, sum, 31);
            s0 += 32;
            mine = at(s0 + lane);
            n = tiles_of(mine);
        }
        if (lane == 0 && (int64_t)p.kv_lens[item.sequence] > (int64_t)p.max_blocks * p.block_size)
            flag_error(p.error_word, p.status, kErrPastCache);
        item.rows = (int)min((int64_t)kTileRows, (int64_t)item.q.q_len * p.group - item.row0);
        // Own keys, counted without the shared prefix, whose rows all see it.
        const int own = item.q.kv_len - p.shared_len;
        const int first = own - item.q.q_len + item.row0 / p.group;
        const int last = own - item.q.q_len + (item.row0 + item.rows - 1) / p.group;
        const int prefix = item.q.prefix - p.shared_len;  // beyond a shared prefix there is none
        item.lo = p.window > 0 && prefix <= 0 ? max(0, first - p.window + 1) : 0;
        item.hi = max(max(0, min(own, last + 1)), prefix);
        item.lo_tile = item.lo / kTileKeys;
        item.shared_tiles = (p.shared_len + kTileKeys - 1) / kTileKeys;
        item.tiles = item.shared_tiles + max(0, (item.hi + kTileKeys - 1) / kTileKeys - item.lo_tile);
    }
    item.first_tile = (int)((int64_t)item.tiles * item.split / t.splits);
    item.tiles = (int)((int64_t)item.tiles * (item.split + 1) / t.splits) - item.first_tile;
    return true;
}

// Tile i of the CTA's walk: its first key and the keys of it that are there to read, in the shared prefix's numbering
// or the sequence's own.
struct TileAt {
    bool shared;
    int32_t t0, lo, hi;
};
__device__ __forceinline__ TileAt tile_at(const AttnParams &p, const Item &item, int i) {
    const int n = item.first_tile + i;
    TileAt at;
    at.shared = n < item.shared_tiles;
    at.t0 = (at.shared ? n : n - item.shared_tiles + item.lo_tile) * kTileKeys;
    at.lo = at.shared ? 0 : item.lo;
    at.hi = at.shared ? p.shared_len : item.hi;
    return at;
}

template <class T, int D, bool MODS>
__global__ void __launch_bounds__(kThreads, 1) attention_tiles(const __grid_constant__ TileParams t) {
    using S = Shape<D>;
    extern __shared__ unsigned char raw[];
    __shared__ __align__(8) uint64_t full[S::kSlots], empty[S::kSlots], queries_in[2], scores[2], weights[2][2], outputs[2],
        drain;
    __shared__ uint32_t tmem_base;
    __shared__ int gave_up;
    __shared__ Item shared_item;
    __shared__ int has_item;
    const AttnParams &p = t.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;  // swizzled tiles start on 1024 bytes
    const uint32_t ring = base + 2 * S::kTileBytes;

    if (tid == 0) {
        gave_up = 0;
        auto init = [](uint64_t *bar, int count) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
        };
        for (int i = 0; i < S::kSlots; ++i) init(&full[i], 1), init(&empty[i], 1);
        for (int i = 0; i < 2; ++i) init(&queries_in[i], 128), init(&scores[i], 1), init(&weights[i][0], 128), init(&weights[i][1], 128), init(&outputs[i], 1);
        init(&drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kIssueWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_base))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        fence_before();
    }
    wait_prerequisites();
    launch_dependents();  // after the wait: what starts now may read all that came before this kernel
    if (warp == 0) {
        Item item;
        const bool found = find_item(t, blockIdx.x, item);
        if (lane == 0) {
            has_item = found;
            if (found) shared_item = item;
        }
    }
    __syncthreads();
    fence_after();
    // All 512 columns there are, so the allocation starts at column 0; the issuing warp counts on it (constants stay out
    // of its way to the tensor cores), which the softmax's addresses make good for the rest.
    const uint32_t tmem = tmem_base;
    const Item &item = shared_item;
    const int n_tiles = has_item ? item.tiles : 0;
    const int active = !has_item ? 0 : item.rows > 128 ? 2 : 1;  // tiles of 128 rows in use

    if (warp < kSoftmaxWarps) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegisters));
        const int g = warp >> 2, row = tid & 127;
        if (g < active) {
            // ---- this thread's row
            const int in_item = g * 128 + row;
            const bool valid = in_item < item.rows;
            const int r = item.row0 + in_item;
            const int token = valid ? r / p.group : 0;
            const int head = item.head * p.group + (valid ? r - token * p.group : 0);
            {
                const uint4 *from = reinterpret_cast<const uint4 *>(
                    p.query + (int64_t)(item.q.q0 + token) * p.q_token_stride + (int64_t)head * p.q_head_stride);
                uint4 v[D / 8];  // all in flight at once
#pragma unroll
                for (int c = 0; c < D / 8; ++c) v[c] = valid ? from[c] : make_uint4(0, 0, 0, 0);
                const uint32_t to = base + g * S::kTileBytes + row * 128;
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    const uint32_t at = to + (c >> 3) * S::kHalfBytes + (((c & 7) ^ (row & 7)) << 4);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v[c].x), "r"(v[c].y),
                                 "r"(v[c].z), "r"(v[c].w)
                                 : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                arrive(smem_u32(&queries_in[g]));
            }
            // What the row sees of its sequence's own keys: [see_lo, see_hi) and everything below see_below.
            int position = 0, see_lo = 0, see_hi = 0, see_below = 0;
            float slope = 0.f;
            if (t.prefix_only) {
                if (MODS && p.slopes && valid) {  // where the row stands behind the prefix
                    int s = token;
                    if (p.q_starts) {
                        int low = 0, high = p.batch;  // the last sequence that starts at or before the token
                        while (high - low > 1) {
                            const int mid = (low + high) / 2;
                            if (p.q_starts[mid] <= token) low = mid;
                            else high = mid;
                        }
                        s = low;
                    }
                    const Sequence q = sequence_of(p, s);
                    position = q.kv_len - q.q_len + token - q.q0;
                }
            } else if (valid) {
                const int own = item.q.kv_len - p.shared_len;
                const int stands = own - item.q.q_len + token;
                see_hi = min(own, stands + 1);
                see_lo = p.window > 0 ? max(0, stands - p.window + 1) : 0;
                see_below = item.q.prefix - p.shared_len;
                position = stands + p.shared_len;
            }
            if (MODS && p.slopes && valid) slope = p.slopes[head] * kLog2e;

            const float scale_log2 = p.scale * kLog2e;
            const float cap_in = p.softcap > 0.f ? scale_log2 * 2.f / p.softcap : 0.f, cap_out = p.softcap * kLog2e;
            const uint32_t s_tmem = tmem + ((uint32_t)(warp & 3) << 21) + g * 128;
            const uint32_t o_tmem = tmem + ((uint32_t)(warp & 3) << 21) + S::kOutColumn + g * D;
            float m = -INFINITY;
            float2 sum = make_float2(0.f, 0.f);
            bool ok = true;
            for (int i = 0; i < n_tiles; ++i) {
                const TileAt at = tile_at(p, item, i);
                if (!warp_waits(smem_u32(&scores[g]), i & 1, &gave_up)) {
                    ok = false;
                    break;
                }
                fence_after();
                // Scores that a mask, cap or bias changes go back to TMEM as they are then.
                const bool sees_all = !valid ? true
                                      : at.shared ? at.t0 + kTileKeys <= p.shared_len
                                                  : (at.t0 >= see_lo && at.t0 + kTileKeys <= see_hi) ||
                                                        at.t0 + kTileKeys <= see_below;
                const bool masked = !__all_sync(~0u, sees_all);
                if (MODS || masked) {
                    const int from = (at.shared ? 0 : see_lo) - at.t0;
                    const int to = (at.shared ? p.shared_len : see_hi) - at.t0;
                    const int below = (at.shared ? 0 : see_below) - at.t0;
                    const float offset = MODS ? (float)((at.shared ? 0 : p.shared_len) + at.t0 - position) : 0.f;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        float y[32];
                        load32(s_tmem + c * 32, y);
                        wait_loads();
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const int k = c * 32 + e;
                            if (MODS) {  // the score times log2(e)
                                // tanh(z) = 1 - 2 / (e^2z + 1), to 2^-22 of the cap, where the exponent's error counts
                                y[e] = p.softcap > 0.f
                                           ? cap_out - 2.f * cap_out * reciprocal_fast(exp2_fast(y[e] * cap_in) + 1.f)
                                           : y[e] * scale_log2;
                                y[e] += slope * (offset + (float)k);
                            }
                            if (masked && !((k >= from && k < to) || k < below)) y[e] = -INFINITY;
                        }
                        store32(s_tmem + c * 32, y);
                    }
                    wait_stores();
                }
                float x[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) load32(s_tmem + c * 32, x[c]);
                wait_loads();
                float tile_top = -INFINITY;
#pragma unroll
                for (int c = 0; c < 4; ++c) tile_top = max_of(tile_top, x[c]);
                const float unit = MODS ? 1.f : scale_log2;
                tile_top *= unit;
                const bool grow = m == -INFINITY ? tile_top > -INFINITY : tile_top > m + kLazy;
                if (__any_sync(~0u, grow)) {
                    const float now = grow ? tile_top : m, factor = grow ? weight_of(m, now) : 1.f;
                    m = now;
                    sum.x *= factor, sum.y *= factor;
                    if (i > 0) {  // the output so far: the products behind it landed before this tile's scores did
#pragma unroll
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t o[16];
                            load16(o_tmem + c * 16, o);
                            wait_loads();
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
                            store16(o_tmem + c * 16, o);
                        }
                    }
                }
                // Values that no row sees (past the length, ahead of the window) may hold anything: 0 times NaN is NaN.
                if (at.t0 < at.lo || at.t0 + kTileKeys > at.hi) {
                    const int slot = (2 * i + 1) % S::kSlots;
                    if (!warp_waits(smem_u32(&full[slot]), ((2 * i + 1) / S::kSlots) & 1, &gave_up)) {
                        ok = false;
                        break;
                    }
                    const int k = at.t0 + row;
                    if (k < at.lo || k >= at.hi) {
#pragma unroll
                        for (int c = 0; c < D / 8; ++c)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                                             ring + slot * S::kTileBytes + (c >> 3) * S::kHalfBytes + row * 128 +
                                             ((c & 7) << 4)),
                                         "r"(0)
                                         : "memory");
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                // The weights, over the scores already read (16 columns for 32 scores), given to the second product in
                // two halves, so that it starts while the second is computed.
                const float2 units = make_float2(unit, unit);
                const float below_zero = m == -INFINITY ? 0.f : -m;
                const float2 references = make_float2(below_zero, below_zero);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t packed[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        float2 w = fma2(make_float2(x[c][e], x[c][e + 1]), units, references);
                        w.x = exp2_fast(w.x);
                        w.y = exp2_fast(w.y);
                        sum = add2(sum, w);
                        packed[e >> 1] = Pack2<T>::of(w.x, w.y);
                    }
                    store16(s_tmem + c * 16, packed);
                    if (c & 1) {
                        wait_stores();
                        fence_before();
                        arrive(smem_u32(&weights[g][c >> 1]));
                    }
                }
            }
            // ---- the row's output
            if (ok && n_tiles > 0) {
                ok = warp_waits(smem_u32(&outputs[g]), 0, &gave_up);
                fence_after();
            }
            if (ok) {
                const float total = sum.x + sum.y;
                const int out_token = item.q.q0 + token;
                const bool partial = t.prefix_only || t.splits > 1;
                const int64_t at = ((int64_t)item.split * p.num_tokens + out_token) * p.q_heads + head;
                const float factor = partial ? 1.f : total == 0.f ? 0.f : 1.f / total;
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    float o[32];
                    if (n_tiles > 0) {
                        load32(o_tmem + c * 32, o);
                        wait_loads();
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0.f;
                    }
                    if (!valid) continue;
                    if (partial) {
                        float4 *to = reinterpret_cast<float4 *>(p.split_o + at * D + c * 32);
#pragma unroll
                        for (int e = 0; e < 8; ++e) to[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                    } else {
                        uint4 *to = reinterpret_cast<uint4 *>(p.out + (int64_t)out_token * p.out_token_stride +
                                                              (int64_t)head * p.out_head_stride + c * 64);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float *v = o + 8 * e;
                            to[e] = make_uint4(Pack2<T>::of(v[0] * factor, v[1] * factor),
                                               Pack2<T>::of(v[2] * factor, v[3] * factor),
                                               Pack2<T>::of(v[4] * factor, v[5] * factor),
                                               Pack2<T>::of(v[6] * factor, v[7] * factor));
                        }
                    }
                }
                if (partial && valid) p.split_ml[at] = make_float2(m, total);
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
    }
    if (warp == kIssueWarp) {
        // The whole warp walks the loop, one elected lane issues: operands then stay in uniform registers. Issued from
        // a divergent branch, a tile's 16 products took 700 cycles longer.
        constexpr uint32_t score_inst = instruction<T>(kTileKeys, false), output_inst = instruction<T>(D, true);
        bool ok = true;
        auto wait = [&](uint64_t *bar, uint32_t parity) {
            if (ok) ok = warp_waits(smem_u32(bar), parity, &gave_up);
            return ok;
        };
        const uint64_t q_operand = operand(base, 16), k_operand = operand(ring, 16),
                       v_operand = operand(ring, S::kHalfBytes);
        auto score = [&](int g, int slot) {
            const uint64_t q = q_operand + (uint32_t)(g * (S::kTileBytes >> 4));
            const uint64_t k = k_operand + (uint32_t)(slot * (S::kTileBytes >> 4));
            if (elect_one()) {
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    constexpr int kHalf = S::kHalfBytes >> 4;
                    const uint32_t step = (c >> 2) * kHalf + (c & 3) * 2;
                    mma_shared(g * 128, q + step, k + step, score_inst, c > 0);
                }
                commit(smem_u32(&scores[g]));
            }
            __syncwarp();
        };
        auto output = [&](int g, int slot, int half, bool accumulate) {
            const uint64_t v = v_operand + (uint32_t)(slot * (S::kTileBytes >> 4) + half * (64 * 128 >> 4));
            if (elect_one()) {
#pragma unroll
                for (int c = 0; c < kTileKeys / 32; ++c)
                    mma_tensor(S::kOutColumn + g * D, g * 128 + half * 32 + c * 8, v + (uint32_t)(c * (16 * 128 >> 4)),
                               output_inst, accumulate || c > 0);
            }
            __syncwarp();
        };
        auto finished = [&](uint64_t *bar) {
            if (elect_one()) commit(smem_u32(bar));
            __syncwarp();
        };
        // Ring order: K 0, V 0, K 1, V 1, ...
        if (n_tiles > 0 && wait(&full[0], 0)) {
            for (int g = 0; g < active; ++g)
                if (wait(&queries_in[g], 0)) {
                    fence_after();
                    score(g, 0);
                }
            finished(&empty[0]);
        }
        int v_slot = 1 % S::kSlots, k_slot = 2 % S::kSlots;
        uint32_t v_phase = 0, k_phase = 0;
        for (int i = 0; ok && i < n_tiles; ++i) {
            const bool more = i + 1 < n_tiles;
            if (!wait(&full[v_slot], v_phase)) break;
            if (more && !wait(&full[k_slot], k_phase)) break;
            for (int g = 0; g < active; ++g) {
                if (!wait(&weights[g][0], i & 1)) break;
                fence_after();
                output(g, v_slot, 0, i > 0);
                if (!wait(&weights[g][1], i & 1)) break;
                fence_after();
                output(g, v_slot, 1, true);
                // The scores land where the weights were: the products execute in the order they are issued.
                if (more) score(g, k_slot);
                else finished(&outputs[g]);
            }
            if (ok) {
                finished(&empty[v_slot]);
                if (more) finished(&empty[k_slot]);
            }
            if ((v_slot += 2) >= S::kSlots) v_slot -= S::kSlots, v_phase ^= 1;
            if ((k_slot += 2) >= S::kSlots) k_slot -= S::kSlots, k_phase ^= 1;
        }
        if (lane == 0) {
            if (!ok) {  // a wait ran out: let what was issued end before TMEM is freed
                commit(smem_u32(&drain));
                const uint64_t deadline = globaltimer() + kWaitNs;
                while (!mbar_try_wait(smem_u32(&drain), 0) && globaltimer() < deadline) {
                }
            }
        }
        __syncwarp();
    } else if (warp == kLoadWarp) {
        // ---- loads: K 0, V 0, K 1, V 1, ... into the ring, one copy of `box` tokens x 64 elements per lane at a time
        const int boxes = kTileKeys / t.box, copies = boxes * S::kHalves;
        int issued = 0;
        bool ok = true;
        for (int n = 0; n < 2 * n_tiles; ++n) {
            const int slot = n % S::kSlots;
            if (n >= S::kSlots &&
                !warp_waits(smem_u32(&empty[slot]), ((n / S::kSlots) & 1) ^ 1, &gave_up)) {
                ok = false;
                break;
            }
            const TileAt at = tile_at(p, item, n / 2);
            const int32_t *table = at.shared ? p.shared_table : p.block_tables + (int64_t)item.sequence * p.table_stride;
            // Up to 32 copies a tile (8-token boxes of 128-wide heads): one per lane.
            const int half = lane / boxes, box = lane - half * boxes;
            const int k = at.t0 + box * t.box;
            const bool wanted = lane < copies && k < at.hi && k + t.box > at.lo;
            int block = 0, in_block = 0;
            if (wanted) {
                const int b = p.block_shift >= 0 ? k >> p.block_shift : k / p.block_size;
                in_block = k - b * p.block_size;
                block = table[b];
                if (block < 0 || block >= p.num_blocks) {
                    flag_error(p.error_word, p.status, kErrPastCache);
                    block = p.num_blocks;  // past the tensor: the copy fills in zeros
                }
            }
            const int count = __popc(__ballot_sync(~0u, wanted));
            const uint32_t bar = smem_u32(&full[slot]);
            if (lane == 0)
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(count * t.box * 128)
                             : "memory");
            __syncwarp();
            if (wanted)
                copy_box(ring + slot * S::kTileBytes + half * S::kHalfBytes + box * t.box * 128,
                         (n & 1) ? &t.values : &t.keys, half * 64, in_block, item.head, block, bar);
            issued = n + 1;
        }
        if (!ok || gave_up) {  // copies may still be landing: give each a bounded wait before the CTA ends
            const uint64_t deadline = globaltimer() + kWaitNs;
            for (int n = max(0, issued - S::kSlots); n < issued; ++n)
                while (!mbar_try_wait(smem_u32(&full[n % S::kSlots]), (n / S::kSlots) & 1) && globaltimer() < deadline) {
                }
        }
        __syncwarp();
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == kIssueWarp)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    if (tid == 0 && gave_up) flag_error(p.error_word, p.status, kErrAttentionWait);
}

// Joins the splits of rows that attention_tiles took, 16 rows per CTA.
constexpr int kJoinRows = 16;
constexpr int kJoinThreads = 128;

template <class T, int D>
__global__ void __launch_bounds__(kJoinThreads) attention_join(const __grid_constant__ TileParams t) {
    __shared__ Item shared_item;
    __shared__ int has_item;
    const AttnParams &p = t.a;
    wait_prerequisites();
    launch_dependents();
    constexpr int kParts = kTileRows / kJoinRows;
    const int part = blockIdx.x % kParts, id = blockIdx.x / kParts;
    if (threadIdx.x < 32) {
        Item item;
        // Item ids count (row tile, split, head); every split holds the same rows.
        const bool found = find_item(t, id / p.kv_heads * p.kv_heads * t.splits + id % p.kv_heads, item);
        if (threadIdx.x == 0) {
            has_item = found;
            if (found) shared_item = item;
        }
    }
    __syncthreads();
    if (!has_item) return;
    const Item &item = shared_item;
    constexpr int kQuads = D / 4;
    const int64_t step = (int64_t)p.num_tokens * p.q_heads;
    for (int k = threadIdx.x; k < kJoinRows * kQuads; k += kJoinThreads) {
        const int in_item = part * kJoinRows + k / kQuads, quad = k % kQuads;
        if (in_item >= item.rows) break;
        const int r = item.row0 + in_item, token = r / p.group;
        const int head = item.head * p.group + r - token * p.group;
        const int64_t at = (int64_t)(item.q.q0 + token) * p.q_heads + head;
        Joined j;
        join_parts(j, t.splits, p.split_ml, p.split_o, kQuads, quad, [&](int i) { return at + i * step; });
        const float inverse = j.sum == 0.f ? 0.f : 1.f / j.sum;
        *reinterpret_cast<uint2 *>(p.out + (int64_t)(item.q.q0 + token) * p.out_token_stride +
                                   (int64_t)head * p.out_head_stride + quad * 8) =
            make_uint2(Pack2<T>::of(j.o.x * inverse, j.o.y * inverse), Pack2<T>::of(j.o.z * inverse, j.o.w * inverse));
    }
}

// ------------------------------------------------------------------------------------------------ host side

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void *sym = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            sym = nullptr;
        return reinterpret_cast<EncodeTiled>(sym);
    }();
    return fn;
}

int make_map(CUtensorMap *map, const AttnParams &p, uint64_t cache, int head_dim, int dtype, int box) {
    EncodeTiled encode = encode_tiled();
    if (!encode) return fail(KVX_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)p.block_size, (cuuint64_t)p.kv_heads,
                                (cuuint64_t)p.num_blocks};
    const cuuint64_t strides[3] = {(cuuint64_t)p.token_stride, (cuuint64_t)p.head_stride, (cuuint64_t)p.block_stride};
    const cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1}, steps[4] = {1, 1, 1, 1};
    const CUresult rc = encode(map, dtype == KVX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                               4, reinterpret_cast<void *>(cache), dims, strides, boxes, steps,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return fail(KVX_ERR_CUDA, "cuTensorMapEncodeTiled failed: %d", (int)rc);
    return KVX_OK;
}

template <class Kernel>
int launch(Kernel kernel, const TileParams &t, int64_t grid, int threads, int smem, cudaStream_t stream) {
    if (grid > 0x7fffffff) return fail(KVX_ERR_INVALID, "more rows than a launch holds");
    cudaLaunchConfig_t cfg = {};
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    KVX_CUDA(cudaLaunchKernelEx(&cfg, kernel, t));
    count_launch();
    return KVX_OK;
}

template <class T, int D>
int launch_typed(const TileParams &t, bool mods, cudaStream_t stream) {
    auto kernel = mods ? attention_tiles<T, D, true> : attention_tiles<T, D, false>;
    KVX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::kBytes));
    const int64_t items = (int64_t)t.row_tiles * t.a.kv_heads;
    if (int rc = launch(kernel, t, items * t.splits, kThreads, Shape<D>::kBytes, stream)) return rc;
    if (t.prefix_only || t.splits == 1) return KVX_OK;
    return launch(attention_join<T, D>, t, items * (kTileRows / kJoinRows), kJoinThreads, 0, stream);
}

}  // namespace

int kvx::tile_box(const AttnParams &p) {
    // A copy lies within one block and fills whole 8-row groups of the swizzle: the block size's largest power of two.
    const int box = std::min(p.block_size & -p.block_size, kTileKeys);
    const bool strides = p.token_stride > 0 && p.head_stride > 0 && p.block_stride > 0 &&
                         std::max({p.token_stride, p.head_stride, p.block_stride}) < (int64_t)1 << 40;
    return box >= 8 && strides && p.num_blocks > 0 ? box : 0;
}

int kvx::launch_tiles(const AttnParams &p, int head_dim, int dtype, bool mods, bool prefix_only, int splits,
                      cudaStream_t stream) {
    TileParams t;
    t.a = p;
    t.box = tile_box(p);
    t.splits = splits;
    t.prefix_only = prefix_only;
    const int64_t rows = (int64_t)p.num_tokens * p.group;
    t.row_tiles = (int)((rows + kTileRows - 1) / kTileRows) + (prefix_only ? 0 : p.batch - 1);
    if (int rc = make_map(&t.keys, p, p.k_cache, head_dim, dtype, t.box)) return rc;
    if (int rc = make_map(&t.values, p, p.v_cache, head_dim, dtype, t.box)) return rc;
    if (head_dim == 128)
        return dtype == KVX_BF16 ? launch_typed<__nv_bfloat16, 128>(t, mods, stream)
                                 : launch_typed<__half, 128>(t, mods, stream);
    return dtype == KVX_BF16 ? launch_typed<__nv_bfloat16, 64>(t, mods, stream)
                             : launch_typed<__half, 64>(t, mods, stream);
}
