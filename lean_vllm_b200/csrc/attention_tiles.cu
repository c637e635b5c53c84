// attention_tiles: up to 256 query rows of one KV head against a stretch of keys, on the 5th-generation tensor cores:
// the form for prompts, drafted tokens in numbers, and a prefix that a whole batch shares, where a key meets so many
// rows that the products bound the time, not the cache.
//
// Work. The query rows of a KV head (its group of heads x the sequence's query tokens, or the whole batch's for a shared
// prefix) share its keys. A CTA takes two tiles of whole tokens, up to 128 rows each, so that one TMA copy brings a
// tile's 64 columns whatever the group (7 heads: 18 tokens, 126 rows), and walks its keys in tiles of 128. For each
// pair of tiles, S = Q K^T and O += P V are one chain of tcgen05.mma each, 128 x 128 x D and 128 x D x 128, with Q, K and
// V in shared memory and S, P and O in TMEM (S, then P in its place, 128 columns a tile; O, D columns a tile).
//
// Where few items would leave SMs idle, for 64-wide heads and behind a shared prefix (kvx_attention's rule), a CTA has one
// tile of rows and an SM two CTAs: one tile's chain of products and softmax alone takes 2900 cycles a tile of keys, and
// would read 22 bytes a cycle, what an SM's share of HBM brings at best.
//
// Roles. One warp copies K and V tiles by TMA into a ring, one copies the queries, one issues the products, one looks up
// what to do next; two groups of 4 warps run the softmax of a tile each, one row per thread. While one tile's scores are
// in the softmax the other's products run, and a CTA takes item after item: the next one's keys and queries arrive and
// its first scores are computed while the last one's output is written. One item per CTA cost 10,000 cycles between two
// items (lookup, queries, first keys, output), a quarter of a prompt of 8192 tokens.
//
// Bound by the tensor cores as the power limit lets them run: a prompt of 8192 tokens of 32 heads over 8, 128 wide, takes
// 458 to 477 us graph-replayed, 1150 to 1200 TFLOP/s, 70 to 73% of a large cuBLAS product's rate, and 510 to 550 called back
// to back, with the clock lower still. A pair of tiles takes 3300 cycles where its products alone
// take 2048: each waits 1250 for the other's (768 of them its own last half and next scores) and spends 2000 in the
// softmax, half of that on the special-function unit. A third of the exponentials on the multiply-add pipe instead made
// that shorter and the whole no faster (498 us); an issuing warp for each tile let both fall into step and contend (499).
//
// The running maximum moves only when a tile's exceeds it by more than 2^8 (kLazy): the weights then stay below 2^8, which
// costs no precision in a floating type, and the accumulated output is rescaled a few times per row, not per tile.

#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "attention.cuh"

namespace {

using namespace kvx;

// Warps of a CTA with GROUPS tiles of rows (two, or one) and CTAS CTAs per SM: the softmax's, then one each that issues
// products, copies keys and values, copies queries and looks up items.
//
// Registers. A row's 128 scores want more than the launch gives each thread, the other warps less. Two tiles, one CTA per
// SM: 256 x 224 + 128 x 56 = 64512, the launch's 384 x 168. One tile, two CTAs: 128 x 200 + 128 x 56 = 32768, 256 x 128;
// one CTA: 128 x 224 + 128 x 56, of the launch's 256 x 224. (128 wide, that is less than ptxas wants: it spills 48 to 64 bytes
// a thread with two tiles, 200 with one tile on each of two CTAs, where an item's end holds all of its output at once.)
template <int GROUPS, int CTAS>
struct Warps {
    static constexpr int kSoftmax = 4 * GROUPS, kIssue = kSoftmax, kLoad = kSoftmax + 1, kQuery = kSoftmax + 2,
                         kPlan = kSoftmax + 3, kThreads = 32 * (kSoftmax + 4);
    static constexpr int kItemReaders = kSoftmax + 3;  // warps that read an item
    static constexpr int kSoftmaxRegisters = CTAS == 1 ? 224 : 200, kOtherRegisters = 56;
    static constexpr int kColumns = 256 * GROUPS;      // of TMEM
};
constexpr float kLazy = 8.f;
constexpr uint64_t kWaitNs = 2000000000ull;  // a wait that has not ended after 2 s is an error

template <int D, int GROUPS, int CTAS>
struct Shape {
    static constexpr int kHalves = D / 64;                      // 128-byte columns of a row
    static constexpr int kTileBytes = kTileKeys * D * 2;        // of 128 rows: queries, keys or values
    static constexpr int kHalfBytes = kTileKeys * 128;
    static constexpr int kSlots = (D == 128 ? 4 : 8) / CTAS;    // ring of K and V tiles: 128 KB an SM
    static constexpr int kStageBytes = 32 * 128;                // of a softmax warp: its rows' output on its way out
    static constexpr int kControlBytes = 1024;                  // barriers and items; the tiles start on 1024 bytes
    static constexpr int kBytes =
        kControlBytes + (GROUPS + kSlots) * kTileBytes + Warps<GROUPS, CTAS>::kSoftmax * kStageBytes;
    static constexpr int kOutColumn = 128 * GROUPS;             // TMEM: S and P of each tile, then O of each
};

struct TileParams {
    AttnParams a;
    CUtensorMap keys, values, queries;
    int32_t tile_tokens;  // query tokens of a tile of up to 128 rows
    int32_t item_tokens;  // and of an item: as many tiles as the CTA has
    int32_t box;          // tokens per copy
    int32_t splits;
    int32_t prefix_only;
    int32_t row_tiles;    // bound on the launch's items per KV head and split
    int32_t *next;        // items given out beyond each CTA's first; 0 between launches
};

struct Item {
    Sequence q;
    int32_t valid;               // 0: no more work
    int32_t sequence, head, token0, tokens, split;  // tokens: of the sequence's (or the batch's) from token0 on
    int32_t lo, hi;              // own keys that any row sees, behind ...
    int32_t front;               // ... those walked first, all rows seeing them: the shared prefix, or the sequence's own one
                                 // where a window leaves keys out behind it
    int32_t front_tiles, tiles;  // their tiles, and all of this split's ...
    int32_t first_tile;          // ... from this one of the item's on
};
static_assert(sizeof(Item) == 64, "four 16-byte reads: with one field more a prompt of 8192 tokens took 553 us, not 537");

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

// 2^x of two values between -127 (0 below) and 60 (2^60 above) on the multiply-add pipe. x = n + f with n the nearest
// integer (left in the low bits by adding 1.5 * 2^23) and f in [-1/2, 1/2]; 2^f by a polynomial with p(0) = 1 whose
// coefficients are a least-maximum fit of the relative error (1e-7); n goes into the exponent. The last product keeps a
// NaN, which the integer addition would turn into a number.
__device__ __forceinline__ float2 exp2_polynomial(float2 x) {
    asm("{\n\tmax.NaN.f32 %0, %0, %1;\n\tmin.NaN.f32 %0, %0, %2;\n\t}" : "+f"(x.x) : "f"(-127.f), "f"(60.f));
    asm("{\n\tmax.NaN.f32 %0, %0, %1;\n\tmin.NaN.f32 %0, %0, %2;\n\t}" : "+f"(x.y) : "f"(-127.f), "f"(60.f));
    const float2 shifted = add2(x, make_float2(12582912.f, 12582912.f));
    const float2 whole = add2(shifted, make_float2(-12582912.f, -12582912.f));
    const float2 f = fma2(whole, make_float2(-1.f, -1.f), x);
    float2 y = fma2(f, make_float2(0.0013264727f, 0.0013264727f), make_float2(0.00967151265f, 0.00967151265f));
    y = fma2(y, f, make_float2(0.0555073374f, 0.0555073374f));
    y = fma2(y, f, make_float2(0.240222421f, 0.240222421f));
    y = fma2(y, f, make_float2(0.693146978f, 0.693146978f));
    y = fma2(y, f, make_float2(1.f, 1.f));
    y = make_float2(__int_as_float(__float_as_int(y.x) + (__float_as_int(shifted.x) << 23)),
                    __int_as_float(__float_as_int(y.y) + (__float_as_int(shifted.y) << 23)));
    return fma2(x, make_float2(0.f, 0.f), y);
}

// Two scores x to cap tanh(x / cap), times log2(e): tanh(z) = 1 - 2 / (e^2z + 1), so that the error is 1e-7 of the cap,
// which is what counts in an exponent. The special-function unit gives 16 results a cycle for the CTA's 32,768 scores a
// pair of tiles, and the weights take one each: the cap takes half a one, a reciprocal for two scores, and has its
// exponential from the polynomial above.
__device__ __forceinline__ void capped(float &x, float &y, float cap_in, float cap_out) {
    const float2 e = exp2_polynomial(mul2(make_float2(x, y), make_float2(cap_in, cap_in)));
    const float2 d = add2(e, make_float2(1.f, 1.f));
    const float r = reciprocal_fast(d.x * d.y) * (-2.f * cap_out);
    const float2 capped = fma2(make_float2(d.y, d.x), make_float2(r, r), make_float2(cap_out, cap_out));
    x = capped.x;
    y = capped.y;
}

// The same for scores within three quarters of the cap, where tanh(z) / z is a polynomial of z^2 (a least-maximum fit of
// the relative error, 3e-8): 7 operations for two scores instead of 25. A tile that no mask touches takes it when all of
// the warp's scores are that small, as scores that a cap only guards are, and caps them on their way into the weights; a
// prompt of 4096 tokens of 32 heads over 8, 128 wide, takes 196 us so and 266 with its scores put back into TMEM capped.
// Elsewhere a chunk of 32 columns does. (A NaN stays one either way.)
struct NearCap {
    float c[6], reach;
    __device__ __forceinline__ NearCap(float scale, float cap) {
        constexpr float kFit[6] = {1.f, -0.333330684f, 0.133265212f, -0.0533902585f, 0.0196649133f, -0.00476949004f};
        const float z = cap > 0.f ? scale / cap : 0.f;  // of a score of 1
        float power = scale * kLog2e;
#pragma unroll
        for (int i = 0; i < 6; ++i, power *= z * z) c[i] = kFit[i] * power;
        reach = z != 0.f ? 0.75f / fabsf(z) : 0.f;
    }
    // Two scores capped, plus `offset`.
    __device__ __forceinline__ float2 cap(float2 v, float2 offset) const {
        const float2 u = mul2(v, v);
        float2 r = fma2(u, make_float2(c[5], c[5]), make_float2(c[4], c[4]));
#pragma unroll
        for (int i = 3; i >= 0; --i) r = fma2(r, u, make_float2(c[i], c[i]));
        return fma2(r, v, offset);
    }
};

// The largest magnitude, NaN aside.
__device__ __forceinline__ float most_of(float most, const float (&x)[32]) {
#pragma unroll
    for (int e = 0; e < 32; e += 2)
        asm("max.f32 %0, %0, %1, %2;" : "+f"(most) : "f"(fabsf(x[e])), "f"(fabsf(x[e + 1])));
    return most;
}

// The lowest n bits, for any n.
__device__ __forceinline__ uint32_t lowest(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1; }

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

// Item `id`: which rows of which sequence, and which keys. Row tiles come last first, since the last ones of a causal
// prompt see the most keys. A whole warp calls this; false: there are no more. `count`: how many there are.
__device__ bool find_item(const TileParams &t, int id, Item &item, int &count) {
    const AttnParams &p = t.a;
    const int lane = threadIdx.x & 31;
    const int per_tile = p.kv_heads * t.splits;
    const int r = id / per_tile;
    item.split = (id - r * per_tile) / p.kv_heads;
    item.head = id - r * per_tile - item.split * p.kv_heads;
    if (t.prefix_only) {
        count = t.row_tiles * per_tile;
        if (id >= count) return false;
        item.sequence = 0;
        item.q = Sequence{0, p.num_tokens, p.shared_len, 0};
        item.token0 = r * t.item_tokens;
        item.tokens = min(t.item_tokens, p.num_tokens - item.token0);
        item.lo = item.hi = 0;
        item.front = p.shared_len;
        item.front_tiles = (p.shared_len + kTileKeys - 1) / kTileKeys;
        item.tiles = item.front_tiles;
    } else {
        auto tiles_of = [&](const Sequence &q) {
            return (int64_t)q.q_len * p.group > p.rows_limit ? (q.q_len + t.item_tokens - 1) / t.item_tokens : 0;
        };
        auto at = [&](int s) { return s < p.batch ? sequence_of(p, s) : Sequence{0, 0, 0, 0}; };
        Sequence mine = at(lane);  // of the 32 sequences looked at now: all there are, often
        int n = tiles_of(mine), total = n;
        for (int s = lane + 32; s < p.batch; s += 32) total += tiles_of(at(s));
        total = __reduce_add_sync(~0u, total);
        count = total * per_tile;
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
                item.token0 = (wanted - before - __shfl_sync(~0u, sum - n, who)) * t.item_tokens;
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
        item.tokens = min(t.item_tokens, item.q.q_len - item.token0);
        // Own keys, counted without the shared prefix, whose rows all see it.
        const int own = item.q.kv_len - p.shared_len;
        const int first = own - item.q.q_len + item.token0, last = first + item.tokens - 1;
        const int prefix = item.q.prefix - p.shared_len;  // beyond a shared prefix there is none
        const int window = window_start(p, first);  // behind the prefix: what lies between may be gone, and is left out
        item.lo = window > prefix ? window : 0;
        item.front = p.shared_len + (window > prefix ? prefix : 0);
        item.hi = max(max(0, min(own, last + 1)), prefix);
        item.front_tiles = (item.front + kTileKeys - 1) / kTileKeys;
        item.tiles = item.front_tiles + max(0, (item.hi + kTileKeys - 1) / kTileKeys - item.lo / kTileKeys);
    }
    item.valid = 1;
    item.first_tile = 0;
    if (t.splits > 1) {  // from tiles * split / splits on, in 32 bits
        const int each = item.tiles / t.splits, rest = item.tiles - each * t.splits;
        auto start_of = [&](int split) { return each * split + rest * split / t.splits; };
        item.first_tile = start_of(item.split);
        item.tiles = start_of(item.split + 1) - item.first_tile;
    }
    return true;
}

// Tile i of the CTA's walk: its first key and the keys of it that are there to read, in the front stretch or behind it (in
// the sequence's own numbering; of a shared prefix, in the prefix's).
struct TileAt {
    bool front;
    int32_t t0, lo, hi;
};
__device__ __forceinline__ TileAt tile_at(const Item &item, int i) {
    const int n = item.first_tile + i;
    TileAt at;
    at.front = n < item.front_tiles;
    at.t0 = (at.front ? n : n - item.front_tiles + item.lo / kTileKeys) * kTileKeys;
    at.lo = at.front ? 0 : item.lo;
    at.hi = at.front ? item.front : item.hi;
    return at;
}

template <int SLOTS>
struct Control {
    uint64_t full[SLOTS], empty[SLOTS];  // ring: filled by copies, read by products
    uint64_t queries_in, queries_read;
    uint64_t scores[2], weights[2][2], outputs[2];  // by tile of 128 rows (and half of its keys)
    uint64_t item_in[2], item_read[2], drain;
    uint32_t tmem_base;
    int gave_up;
    Item items[2];
};

template <class T, int D, int GROUPS, int CTAS, bool MODS>
__global__ void __launch_bounds__(Warps<GROUPS, CTAS>::kThreads, CTAS)
attention_tiles(const __grid_constant__ TileParams t) {
    using S = Shape<D, GROUPS, CTAS>;
    using W = Warps<GROUPS, CTAS>;
    extern __shared__ __align__(1024) unsigned char raw[];
    static_assert(sizeof(Control<S::kSlots>) <= S::kControlBytes, "the control block's room");
    Control<S::kSlots> &control = *reinterpret_cast<Control<S::kSlots> *>(raw);
    auto &full = control.full, &empty = control.empty;
    auto &queries_in = control.queries_in, &queries_read = control.queries_read, &drain = control.drain;
    auto &scores = control.scores, &outputs = control.outputs;
    auto &weights = control.weights;
    auto &item_in = control.item_in, &item_read = control.item_read;
    auto &tmem_base = control.tmem_base;
    int &gave_up = control.gave_up;
    auto &items = control.items;
    const AttnParams &p = t.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = smem_u32(raw) + S::kControlBytes;
    const uint32_t ring = base + GROUPS * S::kTileBytes;

    if (tid == 0) {
        gave_up = 0;
        auto init = [](uint64_t *bar, int count) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
        };
        for (int i = 0; i < S::kSlots; ++i) init(&full[i], 1), init(&empty[i], 1);
        for (int i = 0; i < 2; ++i) {
            init(&scores[i], 1), init(&outputs[i], 1), init(&weights[i][0], 128), init(&weights[i][1], 128);
            init(&item_in[i], 1), init(&item_read[i], W::kItemReaders);
        }
        init(&queries_in, 1), init(&queries_read, 1), init(&drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == W::kIssue) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)),
                     "n"(W::kColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        fence_before();
    }
    __syncthreads();
    fence_after();
    wait_prerequisites();
    launch_dependents();  // after the wait: what starts now may read all that came before this kernel
    // All 512 columns there are start at column 0, a constant that stays out of the products' way.
    const uint32_t tmem = tmem_base;

    // Item n of the CTA, in turn for every warp that reads items; false: there are no more (or a wait ran out).
    auto next_item = [&](int n, Item &item) {
        if (!warp_waits(smem_u32(&item_in[n & 1]), (n >> 1) & 1, &gave_up)) return false;
        item = items[n & 1];
        __syncwarp();
        if (lane == 0) arrive(smem_u32(&item_read[n & 1]));
        return item.valid != 0;
    };
    auto active_of = [&](const Item &item) { return GROUPS == 2 && item.tokens > t.tile_tokens ? 2 : 1; };  // tiles in use

    if (warp < W::kSoftmax) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(W::kSoftmaxRegisters));
        const int g = GROUPS == 2 ? warp >> 2 : 0, row = tid & 127;
        const int row_token = row / p.group, row_head = row - row_token * p.group;
        const uint32_t s_tmem = tmem + ((uint32_t)(warp & 3) << 21) + g * 128;
        const uint32_t o_tmem = tmem + ((uint32_t)(warp & 3) << 21) + S::kOutColumn + g * D;
        const uint32_t stage = ring + S::kSlots * S::kTileBytes + warp * S::kStageBytes;
        const float scale_log2 = p.scale * kLog2e;
        const float cap_in = p.softcap > 0.f ? scale_log2 * 2.f / p.softcap : 0.f, cap_out = p.softcap * kLog2e;
        const NearCap near(MODS ? p.scale : 0.f, MODS ? p.softcap : 0.f);
        uint32_t score_phase = 0, output_phase = 0;
        int ring_at = 0;  // tiles of keys walked before this item
        Item item;
        bool ok = true;
        for (int n = 0; ok && next_item(n, item); ring_at += item.tiles, ++n) {
            if (g >= active_of(item)) continue;
            // ---- this thread's row
            const int in_item = g * t.tile_tokens + row_token;
            const bool valid = row_token < t.tile_tokens && in_item < item.tokens;
            const int token = item.token0 + (valid ? in_item : 0);
            const int head = item.head * p.group + row_head;
            // What the row sees of its sequence's own keys, behind the front stretch if there is one: [see_lo, see_hi) and
            // everything below see_below. (A row that is none sees what is there.)
            int position = 0, see_lo = item.lo, see_hi = item.hi, see_below = 0;
            float slope = 0.f;
            if (t.prefix_only) {
                if (MODS && p.slopes && valid) {  // where the row stands behind the prefix
                    const Sequence q = sequence_of(p, sequence_at(p, token));
                    position = q.kv_len - q.q_len + token - q.q0;
                }
            } else if (valid) {
                const int own = item.q.kv_len - p.shared_len;
                const int stands = own - item.q.q_len + token;
                see_hi = min(own, stands + 1);
                see_lo = window_start(p, stands);
                see_below = item.lo > 0 ? 0 : item.q.prefix - p.shared_len;
                position = stands + p.shared_len;
            }
            if (MODS && p.slopes && valid) slope = p.slopes[head] * kLog2e;

            float m = -INFINITY;
            float2 sum = make_float2(0.f, 0.f);
            // Until a tile is not. (Under a negative scale the capped scores fall as the products rise, and a tile's maximum
            // would be its smallest product: those take the way through TMEM.)
            bool look_near = MODS && p.softcap > 0.f && p.scale > 0.f && !p.slopes;
            // Rows that are none have no say: what is in them is left from before, and the two ways round differently.
            const float reach = valid ? near.reach : INFINITY;
            for (int i = 0; i < item.tiles; ++i) {
                const TileAt at = tile_at(item, i);
                if (!warp_waits(smem_u32(&scores[g]), score_phase, &gave_up)) {
                    ok = false;
                    break;
                }
                score_phase ^= 1;
                fence_after();
                // Scores that a mask, cap or bias changes go back to TMEM as they are then, 32 columns at a time.
                // The modified form asks every row, so that a tile with keys that are not there is masked in every warp; the
                // plain one leaves out rows that are none (each way a prompt is 1% faster, capped or plain).
                const bool sees_all = !MODS && !valid ? true
                                      : at.front ? at.t0 + kTileKeys <= at.hi
                                                 : (at.t0 >= see_lo && at.t0 + kTileKeys <= see_hi) ||
                                                       at.t0 + kTileKeys <= see_below;
                const bool masked = !__all_sync(~0u, sees_all);
                float x[4][32];
                // A cap alone whose scores are near needs no way back through TMEM: the weights' loop below caps them.
                bool near_tile = false;
                if (MODS && look_near && !masked) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) load32(s_tmem + c * 32, x[c]);
                    wait_loads();
                    float most = 0.f;
#pragma unroll
                    for (int c = 0; c < 4; ++c) most = most_of(most, x[c]);
                    near_tile = look_near = __all_sync(~0u, most <= reach);
                }
                if ((MODS || masked) && !near_tile) {
                    int from = (at.front ? 0 : see_lo) - at.t0, to = (at.front ? at.hi : see_hi) - at.t0;
                    int below = (at.front ? 0 : see_below) - at.t0;
                    float offset = MODS ? (float)((at.front ? 0 : p.shared_len) + at.t0 - position) : 0.f;
#pragma unroll 1
                    for (int c = 0; c < 4; ++c, from -= 32, to -= 32, below -= 32, offset += 32.f) {
                        float y[32];
                        load32(s_tmem + c * 32, y);
                        const uint32_t seen = (lowest(to) & ~lowest(from)) | lowest(below);  // by column
                        wait_loads();
                        if (MODS) {  // scores times log2(e)
                            if (p.softcap > 0.f) {
                                if (masked) {  // what is not seen may be NaN, and pairs share a reciprocal
#pragma unroll
                                    for (int e = 0; e < 32; ++e)
                                        if (!(seen >> e & 1)) y[e] = 0.f;
                                }
                                if (__all_sync(~0u, most_of(0.f, y) <= reach)) {
#pragma unroll
                                    for (int e = 0; e < 32; e += 2) {
                                        const float2 v = near.cap(make_float2(y[e], y[e + 1]), make_float2(0.f, 0.f));
                                        y[e] = v.x, y[e + 1] = v.y;
                                    }
                                } else {
#pragma unroll
                                    for (int e = 0; e < 32; e += 2) capped(y[e], y[e + 1], cap_in, cap_out);
                                }
                            } else {
#pragma unroll
                                for (int e = 0; e < 32; ++e) y[e] *= scale_log2;
                            }
                            if (p.slopes) {
#pragma unroll
                                for (int e = 0; e < 32; ++e) y[e] += slope * (offset + (float)e);
                            }
                        }
                        if (masked) {
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (!(seen >> e & 1)) y[e] = -INFINITY;
                        }
                        store32(s_tmem + c * 32, y);
                    }
                    wait_stores();
                }
                if (!near_tile) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) load32(s_tmem + c * 32, x[c]);
                    wait_loads();
                }
                float tile_top = -INFINITY;
#pragma unroll
                for (int c = 0; c < 4; ++c) tile_top = max_of(tile_top, x[c]);
                const float unit = MODS ? 1.f : scale_log2;
                tile_top = near_tile ? near.cap(make_float2(tile_top, tile_top), make_float2(0.f, 0.f)).x : tile_top * unit;
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
                // Values that no row sees (past the length, past a front stretch, ahead of the window) may hold anything: 0
                // times NaN is NaN.
                if ((!MODS || masked) && (at.t0 < at.lo || at.t0 + kTileKeys > at.hi)) {
                    const int copy = 2 * (ring_at + i) + 1, slot = copy % S::kSlots;
                    if (!warp_waits(smem_u32(&full[slot]), (copy / S::kSlots) & 1, &gave_up)) {
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
                auto weigh = [&](auto exponent) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t packed[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float2 w = exponent(make_float2(x[c][e], x[c][e + 1]));
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
                };
                if (MODS && near_tile) weigh([&](float2 v) { return near.cap(v, references); });
                else weigh([&](float2 v) { return fma2(v, units, references); });
            }
            // ---- the row's output
            if (ok && item.tiles > 0) {
                ok = warp_waits(smem_u32(&outputs[g]), output_phase, &gave_up);
                output_phase ^= 1;
                fence_after();
            }
            if (!ok) break;
            const float total = sum.x + sum.y;
            const bool partial = t.prefix_only || t.splits > 1;
            const float factor = partial ? 1.f : total == 0.f ? 0.f : 1.f / total;
            // 128 bytes of each of the warp's 32 rows at a time go through shared memory, so that they leave in whole
            // lines: 32 partial ones or 64 finished ones.
            auto staged = [&](int chunk) { return stage + lane * 128 + ((chunk ^ (lane & 7)) << 4); };
            auto write_out = [&](uint64_t to, int64_t byte) {  // `to`: this thread's row
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 8; ++k) {  // 4 rows of 8 chunks at once
                    const int from_row = 4 * k + (lane >> 3), chunk = lane & 7;
                    const uint64_t at = __shfl_sync(~0u, to, from_row);
                    uint4 v;
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                                 : "r"(stage + from_row * 128 + ((chunk ^ (from_row & 7)) << 4)));
                    if (at) *reinterpret_cast<uint4 *>(at + byte + chunk * 16) = v;
                }
                __syncwarp();
            };
            const int out_token = item.q.q0 + token;
            const int64_t split_row = ((int64_t)item.split * p.num_tokens + out_token) * p.q_heads + head;
            uint64_t to = 0;
            if (valid)
                to = partial ? reinterpret_cast<uint64_t>(p.split_o + split_row * D)
                             : p.out + (int64_t)out_token * p.out_token_stride + (int64_t)head * p.out_head_stride;
            float all[D / 32][32];
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                if (item.tiles > 0) {
                    load32(o_tmem + c * 32, all[c]);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) all[c][e] = 0.f;
                }
            }
            wait_loads();
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                const float(&o)[32] = all[c];
                if (partial) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(staged(e)), "f"(o[4 * e]),
                                     "f"(o[4 * e + 1]), "f"(o[4 * e + 2]), "f"(o[4 * e + 3])
                                     : "memory");
                    write_out(to, c * 128);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float *v = o + 8 * e;
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(staged((c & 1) * 4 + e)),
                                     "r"(Pack2<T>::of(v[0] * factor, v[1] * factor)),
                                     "r"(Pack2<T>::of(v[2] * factor, v[3] * factor)),
                                     "r"(Pack2<T>::of(v[4] * factor, v[5] * factor)),
                                     "r"(Pack2<T>::of(v[6] * factor, v[7] * factor))
                                     : "memory");
                    }
                    if (c & 1) write_out(to, (c >> 1) * 128);
                }
            }
            if (partial && valid) p.split_ml[split_row] = make_float2(m, total);
            fence_before();  // the next item's first product overwrites what was read
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(W::kOtherRegisters));
    }
    if (warp == W::kIssue) {
        // The whole warp walks the loop, one elected lane issues: operands then stay in uniform registers. Issued from
        // a divergent branch, a tile's 16 products took 700 cycles longer.
        constexpr uint32_t score_inst = instruction<T>(kTileKeys, false), output_inst = instruction<T>(D, true);
        bool ok = true;
        auto wait = [&](uint64_t *bar, uint32_t parity) {
            if (ok) ok = warp_waits(smem_u32(bar), parity, &gave_up);
            return ok;
        };
        const uint32_t columns = GROUPS == 2 ? 0 : tmem;
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
                    mma_shared(columns + g * 128, q + step, k + step, score_inst, c > 0);
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
                    mma_tensor(columns + S::kOutColumn + g * D, columns + g * 128 + half * 32 + c * 8,
                               v + (uint32_t)(c * (16 * 128 >> 4)), output_inst, accumulate || c > 0);
            }
            __syncwarp();
        };
        auto finished = [&](uint64_t *bar) {
            if (elect_one()) commit(smem_u32(bar));
            __syncwarp();
        };
        // The ring holds K 0, V 0, K 1, V 1, ... of item after item.
        int k_slot = 0, v_slot = 1;
        uint32_t ring_phase[2] = {0, 0};  // of the K and the V copy that come next
        uint32_t weight_phase[2] = {0, 0}, query_phase = 0;
        auto advance = [&](int &slot, uint32_t &phase) {
            if ((slot += 2) >= S::kSlots) slot -= S::kSlots, phase ^= 1;
        };
        Item item;
        for (int n = 0; ok && next_item(n, item); ++n) {
            const int active = active_of(item);
            if (item.tiles == 0) continue;
            if (!wait(&queries_in, query_phase) || !wait(&full[k_slot], ring_phase[0])) break;
            query_phase ^= 1;
            fence_after();
            // A tile's first scores land where the last item's weights were, behind the product that read them.
            for (int g = 0; g < active; ++g) score(g, k_slot);
            finished(&empty[k_slot]);
            if (item.tiles == 1) finished(&queries_read);
            advance(k_slot, ring_phase[0]);
            for (int i = 0; ok && i < item.tiles; ++i) {
                const bool more = i + 1 < item.tiles;
                if (!wait(&full[v_slot], ring_phase[1])) break;
                for (int g = 0; g < active; ++g) {
                    if (!wait(&weights[g][0], weight_phase[g])) break;
                    fence_after();
                    output(g, v_slot, 0, i > 0);
                    if (more && g == 0 && !wait(&full[k_slot], ring_phase[0])) break;
                    if (!wait(&weights[g][1], weight_phase[g])) break;
                    weight_phase[g] ^= 1;
                    fence_after();
                    output(g, v_slot, 1, true);
                    // The scores land where the weights were: the products execute in the order they are issued.
                    if (!more) finished(&outputs[g]);
                    else score(g, k_slot);
                }
                if (!ok) break;
                finished(&empty[v_slot]);
                advance(v_slot, ring_phase[1]);
                if (more) {
                    finished(&empty[k_slot]);
                    if (i + 2 == item.tiles) finished(&queries_read);
                    advance(k_slot, ring_phase[0]);
                }
            }
        }
        if (!ok) {  // a wait ran out: let what was issued end before TMEM is freed
            finished(&drain);
            const uint64_t deadline = globaltimer() + kWaitNs;
            while (!mbar_try_wait(smem_u32(&drain), 0) && globaltimer() < deadline) {
            }
        }
        __syncwarp();
    } else if (warp == W::kLoad) {
        // ---- K 0, V 0, K 1, V 1, ... into the ring, one copy of `box` tokens x 64 elements per lane
        const int boxes = kTileKeys / t.box, copies = boxes * S::kHalves;  // at most 32: 8-token boxes, 128-wide heads
        const int half = lane / boxes, box = lane - half * boxes;
        int issued = 0;
        bool ok = true;
        Item item;
        for (int n = 0; ok && next_item(n, item); ++n) {
            const int32_t *own_table = p.block_tables + (int64_t)item.sequence * p.table_stride;
            const int32_t *front_table = p.shared_len > 0 ? p.shared_table : own_table;
            for (int i = 0; ok && i < item.tiles; ++i) {
                const TileAt at = tile_at(item, i);
                const int k = at.t0 + box * t.box;
                const bool wanted = lane < copies && k < at.hi && k + t.box > at.lo;
                int block = 0, in_block = 0;
                if (wanted) {
                    const int b = p.block_shift >= 0 ? k >> p.block_shift : k / p.block_size;
                    in_block = k - b * p.block_size;
                    block = (at.front ? front_table : own_table)[b];
                    if (block < 0 || block >= p.num_blocks) {
                        flag_error(p.error_word, p.status, kErrPastCache);
                        block = p.num_blocks;  // past the tensor: the copy fills in zeros
                    }
                }
                const int bytes = __popc(__ballot_sync(~0u, wanted)) * t.box * 128;
                for (int kv = 0; kv < 2; ++kv, ++issued) {
                    const int slot = issued % S::kSlots;
                    if (issued >= S::kSlots &&
                        !warp_waits(smem_u32(&empty[slot]), ((issued / S::kSlots) & 1) ^ 1, &gave_up)) {
                        ok = false;
                        break;
                    }
                    const uint32_t bar = smem_u32(&full[slot]);
                    if (lane == 0)
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
                                     : "memory");
                    __syncwarp();
                    if (wanted)
                        copy_box(ring + slot * S::kTileBytes + half * S::kHalfBytes + box * t.box * 128,
                                 kv ? &t.values : &t.keys, half * 64, in_block, item.head, block, bar);
                }
            }
        }
        // Copies that nobody waited for (a wait ran out) may still be landing: give each a bounded wait.
        __syncwarp();
        if (*(volatile int *)&gave_up) {
            const uint64_t deadline = globaltimer() + kWaitNs;
            for (int c = max(0, issued - S::kSlots); c < issued; ++c)
                while (!mbar_try_wait(smem_u32(&full[c % S::kSlots]), (c / S::kSlots) & 1) && globaltimer() < deadline) {
                }
        }
        __syncwarp();
    } else if (warp == W::kQuery) {
        // ---- query rows: one copy per tile and 64 columns. Rows past the tokens there are come as zeros or as the next
        // sequence's, those past a tile's whole tokens as whatever was there: each row's scores are its own.
        const int bytes = t.tile_tokens * p.group * 128;  // of a copy
        uint32_t read_phase = 0;
        bool waiting = false;  // for the products that read the queries before
        Item item;
        for (int n = 0; next_item(n, item); ++n) {
            if (item.tiles == 0) continue;  // nothing reads them
            if (waiting && !warp_waits(smem_u32(&queries_read), read_phase, &gave_up)) break;
            if (waiting) read_phase ^= 1;
            waiting = true;
            const int copies = active_of(item) * S::kHalves;
            const uint32_t bar = smem_u32(&queries_in);
            if (lane == 0)
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(copies * bytes)
                             : "memory");
            __syncwarp();
            if (lane < copies) {
                const int g = lane / S::kHalves, half = lane % S::kHalves;
                asm volatile(
                    "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
                    "%4}], [%5];" ::"r"(base + g * S::kTileBytes + half * S::kHalfBytes),
                    "l"(&t.queries), "r"(half * 64), "r"(item.head * p.group),
                    "r"(item.q.q0 + item.token0 + g * t.tile_tokens), "r"(bar)
                    : "memory");
            }
        }
        if (*(volatile int *)&gave_up && waiting) {  // a copy may still be landing
            const uint64_t deadline = globaltimer() + kWaitNs;
            while (!mbar_try_wait(smem_u32(&queries_in), read_phase) && globaltimer() < deadline) {
            }
        }
        __syncwarp();
    } else if (warp == W::kPlan) {
        // ---- what to do: the CTA's first item by its number, then whichever is next
        int id = blockIdx.x;
        for (int n = 0;; ++n) {
            Item item;
            int count = 0;
            item.valid = 0;
            const bool found = find_item(t, id, item, count);
            if (n >= 2 && !warp_waits(smem_u32(&item_read[n & 1]), ((n >> 1) & 1) ^ 1, &gave_up)) break;
            if (lane == 0) {
                items[n & 1] = item;
                if (!found) items[n & 1].valid = 0;
                arrive(smem_u32(&item_in[n & 1]));
                if (found) {
                    id = gridDim.x + atomicAdd(t.next, 1);
                    // One draw per item: the last of all puts the counter back.
                    if (id - (int)gridDim.x == count - 1) *t.next = 0;
                }
            }
            __syncwarp();
            if (!found) break;
            id = __shfl_sync(~0u, id, 0);
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == W::kIssue)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(W::kColumns) : "memory");
    if (tid == 0 && gave_up) flag_error(p.error_word, p.status, kErrAttentionWait);
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

int encode(CUtensorMap *map, int rank, uint64_t address, int dtype, const cuuint64_t *dims, const cuuint64_t *strides,
           const cuuint32_t *box) {
    EncodeTiled fn = encode_tiled();
    if (!fn) return fail(KVX_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    const cuuint32_t steps[4] = {1, 1, 1, 1};
    const CUresult rc = fn(map, dtype == KVX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                           rank, reinterpret_cast<void *>(address), dims, strides, box, steps,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) return fail(KVX_ERR_CUDA, "cuTensorMapEncodeTiled failed: %d", (int)rc);
    return KVX_OK;
}

// A cache by (element, token of a block, head, block), copied 64 elements of `box` tokens at a time.
int cache_map(CUtensorMap *map, const AttnParams &p, uint64_t cache, int head_dim, int dtype, int box) {
    const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)p.block_size, (cuuint64_t)p.kv_heads,
                                (cuuint64_t)p.num_blocks};
    const cuuint64_t strides[3] = {(cuuint64_t)p.token_stride, (cuuint64_t)p.head_stride, (cuuint64_t)p.block_stride};
    const cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1};
    return encode(map, 4, cache, dtype, dims, strides, boxes);
}

// The queries by (element, head, token), copied 64 elements of a KV head's group and some tokens at a time.
int query_map(CUtensorMap *map, const AttnParams &p, int head_dim, int dtype, int tokens) {
    const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)p.q_heads, (cuuint64_t)p.num_tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)p.q_head_stride, (cuuint64_t)p.q_token_stride};
    const cuuint32_t boxes[3] = {64, (cuuint32_t)p.group, (cuuint32_t)tokens};
    return encode(map, 3, p.query, dtype, dims, strides, boxes);
}

template <class T, int D, int GROUPS, int CTAS, bool MODS>
int launch_typed(const TileParams &t, const Device &device, const Queue &queue) {
    static AllowedSmem allowed;
    auto kernel = attention_tiles<T, D, GROUPS, CTAS, MODS>;
    using S = Shape<D, GROUPS, CTAS>;
    if (int rc = allowed.allow(kernel, S::kBytes, device.index)) return rc;
    // One wave of CTAs, each taking item after item.
    const int64_t items = (int64_t)t.row_tiles * t.a.kv_heads * t.splits;
    const int64_t grid = std::min<int64_t>(items, (int64_t)device.sms * CTAS);
    return launch(kernel, grid, Warps<GROUPS, CTAS>::kThreads, S::kBytes, queue, t);
}

template <class T, int D>
int launch_typed(const TileParams &t, int groups, bool mods, const Device &device, const Queue &queue) {
    if constexpr (D == 128) {
        if (groups == 2)
            return mods ? launch_typed<T, D, 2, 1, true>(t, device, queue) : launch_typed<T, D, 2, 1, false>(t, device, queue);
        // No more items than SMs: a CTA has an SM, and twice the ring, to itself. A prompt of 256 tokens of 32 heads over 8
        // takes 9.5 us so and 10.3 in the other shape, one of 512 12.9 and 14.2 (64 wide: 8.2 and 8.2, 10.7 and 11.1).
        // Behind a shared prefix two CTAs per SM are ahead: 64 requests behind 8192 tokens take 37.7 us so and 39.9 in this
        // shape, 5 of 4 drafts behind 30,011 44.4 and 49.0.
        if (!t.prefix_only && (int64_t)t.row_tiles * t.a.kv_heads * t.splits <= device.sms)
            return mods ? launch_typed<T, D, 1, 1, true>(t, device, queue) : launch_typed<T, D, 1, 1, false>(t, device, queue);
    }
    return mods ? launch_typed<T, D, 1, 2, true>(t, device, queue) : launch_typed<T, D, 1, 2, false>(t, device, queue);
}

}  // namespace

int kvx::tile_box(const AttnParams &p) {
    // A copy lies within one block and fills whole 8-row groups of the swizzle: the block size's largest power of two.
    const int box = std::min(p.block_size & -p.block_size, kTileKeys);
    bool strides = p.group <= 128;  // a token's rows fit a tile
    for (int64_t stride : {p.token_stride, p.head_stride, p.block_stride, p.q_head_stride, p.q_token_stride})
        strides = strides && stride > 0 && stride < (int64_t)1 << 40;
    return box >= 8 && strides && p.num_blocks > 0 ? box : 0;
}

int kvx::launch_tiles(const AttnParams &p, int head_dim, int dtype, bool mods, bool prefix_only, int groups,
                      int splits, const Device &device, const Queue &queue) {
    TileParams t;
    t.a = p;
    t.box = tile_box(p);
    t.splits = splits;
    t.prefix_only = prefix_only;
    t.next = p.counters + kTileCounter;
    t.tile_tokens = 128 / p.group;
    t.item_tokens = groups * t.tile_tokens;
    t.row_tiles = (p.num_tokens + t.item_tokens - 1) / t.item_tokens + (prefix_only ? 0 : p.batch - 1);
    if (int rc = cache_map(&t.keys, p, p.k_cache, head_dim, dtype, t.box)) return rc;
    if (int rc = cache_map(&t.values, p, p.v_cache, head_dim, dtype, t.box)) return rc;
    if (int rc = query_map(&t.queries, p, head_dim, dtype, t.tile_tokens)) return rc;
    if (head_dim == 128)
        return dtype == KVX_BF16 ? launch_typed<__nv_bfloat16, 128>(t, groups, mods, device, queue)
                                 : launch_typed<__half, 128>(t, groups, mods, device, queue);
    return dtype == KVX_BF16 ? launch_typed<__nv_bfloat16, 64>(t, groups, mods, device, queue)
                             : launch_typed<__half, 64>(t, groups, mods, device, queue);
}
