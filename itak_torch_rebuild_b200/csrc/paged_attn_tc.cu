// Attention of a ragged batch over the pages of its sequences on the 5th-generation tensor cores, for calls with many
// (row, head) pairs per KV head: prompt chunks, and verify blocks beyond the streaming kernel's 16 pairs.
//
//   S = Q K^T,  P = 2^(c S - m),  O += P V,  out = O / sum P,   c = scale * log2(e), one pass over the keys (P times a
//   constant where the pages are halfs, see kLift).
//
// A cell is (sequence, KV head, block of 256 pairs); a pair is a query row and one of the heads of the KV head's group, so
// that all heads of a group share the K and V tiles.  One CTA per SM walks an equal, contiguous run of the launch's
// 128-key tiles laid end to end over all cells; a cell cut by the end of a run leaves a partial (maximum, sum, output), and
// the CTA that takes the cell's last ticket joins them.  No CTA waits for another.
//
// Two streams keep the tensor core busy while a softmax runs: stream i has 128 accumulator rows (tensor-memory lanes), a
// warpgroup whose thread r owns row r, and its own S and O in tensor memory:
//   columns   0-127  S0, then in place its weights P0       columns 256-...  O0
//   columns 128-255  S1, then P1                            columns 256 + D  O1
//   more than 128 pairs: stream i holds pairs [128 i, 128 i + 128) of the block and takes every tile it sees;
//   128 pairs or fewer ("twin"): both hold the same pairs, stream i takes every second tile, and the two are joined at the
//                        end - otherwise tensor core and loads would wait for one softmax after every tile.
// One thread per stream issues its products, O += P V(t) and then S = Q K(t + 1), and the two take turns; a thread's products
// complete in order, so S may overwrite the weights of the tile before without a barrier of its own, and scores that are
// complete vouch for every product issued before them.
//
// Warps 0-3 and 4-7: softmax of stream 0 and 1.  Warps 8 and 10: their products (one lane each); 8 allocates tensor memory.
// Warp 9: TMA loads of K and V through one ring, K(t), V(t), K(t + 1), ...; a tile is fetched page by page, lane j taking one
// box (64 channels of the rows that a page has in the tile), pages outside the keys of the block left out.  Score columns of
// keys that a row does not see become -infinity whatever the tile holds there; V rows outside the block's keys are
// overwritten with zeros in shared memory, since a weight of zero does not hide a NaN.
//
// 16-bit rows: products are exact, weights are rounded to the pages' type (half a step of the output's type, averaged over
// the keys).  f32 rows: x = h + l with two halfs for queries and weights, twice the products, f32-grade results.
//
// The accumulator is rescaled in tensor memory only when a row's maximum grows by more than 2^8; until then the old
// maximum is used for weights and sum alike, so nothing is lost.
//
// Bound: a 128 x 128 tile of both products takes 1024 clocks on the tensor core (D = 128) and its 16384 exponentials 1024
// clocks on the special-function units.  A round (both products of a tile of one stream) takes about 1600: softmax and
// products of one stream follow one another, and two streams do not quite cover that chain.  (2^x by a polynomial on the
// multiply-add pipe for part of the weights made it longer.)  Measured: 4096 bf16 rows at 16384 keys, 32 / 8 heads of 128:
// 956 us (826 before the power limit sets in), 1.01 PFLOP/s of 1.66; 4 x 512 rows at 1024-2048 keys: f16 73 us, f32 153 us,
// where a cell's end (3 tiles' time), the joins and 14000 clocks before the first tile count as much as the tiles.
#include <cuda.h>

#include <type_traits>

#include "attn_common.cuh"
#include "paged.cuh"
#include "tcgen05.cuh"

namespace itk {
namespace paged {
namespace {

constexpr int kThreads = 384;  // two warpgroups of softmax, and one of product, load and two idle warps
constexpr int kMmaWarp = 8, kLoadWarp = 9;  // stream i's products: warp kMmaWarp + 2 i
// Registers: the softmax threads hold a whole row of scores.  setmaxnreg moves registers between the warpgroups of a
// block launched with kLaunchRegs a thread: 256 x 216 + 128 x 72 = 384 x 168.
constexpr int kLaunchRegs = 168, kSoftmaxRegs = 216, kOtherRegs = 72;
static_assert(256 * kSoftmaxRegs + 128 * kOtherRegs <= kThreads * kLaunchRegs, "registers of the block");
constexpr uint32_t kTile = 128;       // keys of a tile, and rows of a stream
constexpr uint32_t kBlockPairs = 256;
constexpr uint32_t kTmemCols = 512, kTmemO = 256;
constexpr float kRescaleStep = 8.f;
// How the tiles of all cells are cut into runs.  A cell's end costs its CTA about 3 tiles (the last products, the rows' way
// out, the next queries), so each cell reserves as many beyond its own; a cut inside a cell costs two CTAs a partial each and
// one of them the join; a cut that would leave kSnap tiles at a cell's beginning or end moves there.
constexpr uint32_t kCellCost = 3, kSnap = 1;
constexpr uint32_t kSmemBytes = 232448;   // all that a block can have
constexpr uint32_t kTailBytes = 3u << 10;    // mbarriers, the roles' items, the streams' exchange
constexpr long long kRestClocks = 2000000000ll;  // about a second, for what is in flight to come to rest when a call ends early

template <typename T>
struct RowTraits;
template <>
struct RowTraits<float> {
    using Page = __half;
    static constexpr bool kSplit = true;
};
template <>
struct RowTraits<__half> {
    using Page = __half;
    static constexpr bool kSplit = false;
};
template <>
struct RowTraits<__nv_bfloat16> {
    using Page = __nv_bfloat16;
    static constexpr bool kSplit = false;
};

template <typename T, int D>
struct Shape {
    static constexpr bool kSplit = RowTraits<T>::kSplit;
    static constexpr uint32_t kPanel = kTile * 128;              // bytes of [128 rows][64 channels]
    static constexpr uint32_t kStage = (D / 64) * kPanel;        // a K or V tile
    static constexpr uint32_t kQ = (kSplit ? 2 : 1) * kStage;    // a stream's queries: (high) panels, then low ones
    static constexpr uint32_t kStages = (kSmemBytes - kTailBytes - 2 * kQ) / kStage;
    static constexpr uint32_t kSmem = 2 * kQ + kStages * kStage + kTailBytes;
    static_assert(kStages >= 3, "K(t), V(t) and K(t + 1)");
    static_assert(kStages * kStage >= (2 * kMaxSeqs + 1) * 8 + kMaxSeqs * 12, "the ring is the planning's scratch");
};

struct SeqInfo {
    uint32_t row0, rows, len;  // len: as stated; there are min(len, room) keys
};

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t channel, int32_t row, int32_t head,
                                         int32_t page) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];\n" ::"r"(dst),
        "l"(map), "r"(bar), "r"(channel), "r"(row), "r"(head), "r"(page)
        : "memory");
}
__device__ __forceinline__ void both_sync() { asm volatile("bar.sync 1, 256;\n" ::: "memory"); }

__device__ __forceinline__ uint32_t pack2(__half, float x, float y) {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16, float x, float y) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// Two f32 values in one 64-bit register: the packed forms do two multiply-adds or sums in one issue.
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN when one of them is
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// The keys that pairs [p0, p1) of a sequence see, and the 128-key tiles that hold them (none: t0 == t1).
struct KeyRange {
    uint32_t lo, hi, t0, t1;
};
__device__ __forceinline__ KeyRange keys_of(const SeqInfo& q, uint32_t p0, uint32_t p1, uint32_t group, uint32_t window, uint32_t room) {
    const int32_t pos0 = static_cast<int32_t>(q.len) - static_cast<int32_t>(q.rows);
    const int32_t first = pos0 + static_cast<int32_t>(p0 / group), last = pos0 + static_cast<int32_t>((p1 - 1) / group);
    KeyRange r;
    r.hi = last >= 0 ? min(static_cast<uint32_t>(last) + 1u, room) : 0u;
    r.lo = window != 0 && first >= 0 && static_cast<uint32_t>(first) >= window ? first + 1 - window : 0u;
    if (r.lo >= r.hi) r.lo = r.hi = 0;
    r.t0 = r.lo / kTile;
    r.t1 = (r.hi + kTile - 1) / kTile;
    return r;
}
// Tiles a cell takes in a run: at least one, so that a block that sees nothing is still written.
__device__ __forceinline__ uint32_t cell_tiles(const SeqInfo& q, uint32_t block, uint32_t group, uint32_t window, uint32_t room) {
    const KeyRange r = keys_of(q, block * kBlockPairs, min(q.rows * group, (block + 1) * kBlockPairs), group, window, room);
    return max(r.t1 - r.t0, 1u);
}

// One cell, or the part of one that falls into this CTA's run.  Each role (loads, products, softmax) walks the run with an
// item of its own in shared memory: a dozen of registers less in every thread.
struct Item {
    SeqInfo q;
    uint32_t s, kvh, block, blocks, pairs;  // pairs of the block
    uint32_t T, off, n;                     // tiles of the cell, and of those this CTA's [off, off + n)
    uint32_t twin;                          // both streams hold the same pairs
    uint32_t lo, hi;                        // keys of the block
    uint32_t t0, t1;                        // tiles to load
    uint32_t a[2], e[2];                    // stream i: tiles a[i], a[i] + step, ... below e[i]
    uint32_t step;
    uint32_t more;  // the run goes on
    uint64_t pos;   // of tile `off` in the launch's order
};
struct Run {
    const AttnParams& p;
    uint64_t end;
    uint32_t room;

    __device__ __forceinline__ void open_seq(Item& it) const {
        Batch b = p.batch;
        b.status = nullptr;
        const Seq q = seq_of(b, it.s, p.pool.page_shift);
        it.q = SeqInfo{q.row0, q.rows, q.len};
        it.blocks = (it.q.rows * p.group + kBlockPairs - 1) / kBlockPairs;
    }
    __device__ __forceinline__ void open_cell(Item& it, uint32_t off) const {
        const uint32_t all = it.q.rows * p.group, p0 = it.block * kBlockPairs, p1 = min(all, p0 + kBlockPairs);
        it.pairs = p1 - p0;
        it.twin = it.pairs <= kTile ? 1u : 0u;
        const KeyRange r = keys_of(it.q, p0, p1, p.group, p.window, room);
        it.T = max(r.t1 - r.t0, 1u);
        it.off = off;
        it.n = static_cast<uint32_t>(min(end - it.pos, static_cast<uint64_t>(it.T - off)));
        it.lo = r.lo;
        it.hi = r.hi;
        it.t0 = min(r.t0 + off, r.t1);
        it.t1 = min(it.t0 + it.n, r.t1);
        if (it.twin) {
            it.step = 2;
            it.a[0] = it.t0;
            it.a[1] = it.t0 + 1;
            it.e[0] = it.e[1] = it.t1;
        } else {
            it.step = 1;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const KeyRange k = keys_of(it.q, p0 + i * kTile, i == 0 ? p0 + kTile : p1, p.group, p.window, room);
                it.a[i] = max(it.t0, k.t0);
                it.e[i] = min(it.t1, k.t1);
            }
        }
        it.more = 1;
    }
    __device__ __forceinline__ void next(Item& it) const {
        it.pos += it.T + kCellCost - it.off;
        it.more = 0;
        if (it.pos >= end) return;
        if (++it.block == it.blocks) {
            it.block = 0;
            if (++it.kvh == p.pool.kv_heads) {
                it.kvh = 0;
                do {  // a sequence with rows follows, since the launch has tiles left
                    if (++it.s >= p.batch.n_seqs) return;
                    open_seq(it);
                } while (it.blocks == 0);
            }
        }
        open_cell(it, 0);
    }
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) paged_tc_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap kmap,
                                                               const __grid_constant__ CUtensorMap vmap) {
    using P = typename RowTraits<T>::Page;
    using Sh = Shape<T, D>;
    constexpr bool SPLIT = Sh::kSplit;
    constexpr uint32_t NST = Sh::kStages;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* const smem = smem_raw;
    if ((smem_u32(smem) & 1023u) != 0) {  // (the tiles' swizzle goes by address bits; never so far)
        after_predecessor();
        if (threadIdx.x == 0) raise(p.batch, kWaitRanOut);
        const uint32_t rows = min(p.batch.row_start[p.batch.n_seqs], p.batch.total_rows);
        for (uint32_t row = blockIdx.x; row < rows; row += gridDim.x) {
            for (uint32_t c = threadIdx.x; c < p.q_heads * p.pool.head_dim; c += kThreads) static_cast<T*>(p.out)[row * p.out_row + c] = from_f32<T>(NAN);
            if (p.lse)
                for (uint32_t h = threadIdx.x; h < p.q_heads; h += kThreads) p.lse[static_cast<uint64_t>(row) * p.q_heads + h] = NAN;
        }
        return;
    }
    const uint32_t qbuf = smem_u32(smem), ring = qbuf + 2 * Sh::kQ, tail = ring + NST * Sh::kStage;
    unsigned char* const tail_ptr = smem + 2 * Sh::kQ + NST * Sh::kStage;
    // mbarriers
    const uint32_t bar_full = tail;                // [stage] the tile has landed
    const uint32_t bar_empty = bar_full + 8 * NST;  // [stage] every product that reads it is complete
    const uint32_t bar_s = bar_empty + 8 * NST;     // [stream] scores complete
    const uint32_t bar_p = bar_s + 16;              // [stream][half] the weights of half of the tile's keys are stored
    const uint32_t bar_o = bar_p + 32;              // [stream] the cell's last product complete
    const uint32_t bar_q = bar_o + 16;              // [stream] the cell's queries are in shared memory
    const uint32_t bar_land = bar_q + 16;           // a V tile that needs zero rows has landed
    const uint32_t bar_done = bar_land + 8;         // everything issued to the tensor core is complete
    const uint32_t bar_t = bar_done + 8;            // [stream] the products' thread has come to the cell
    constexpr uint32_t kWordAt = 16 * NST + 112, kItemsAt = kWordAt + 24, kItems = 7;
    static_assert(kItemsAt + kItems * sizeof(Item) + 256 * sizeof(float2) <= kTailBytes, "tail");
    uint32_t* const word = reinterpret_cast<uint32_t*>(tail_ptr + kWordAt);  // [0] tensor memory, [1] joined flag
    volatile uint32_t* const abort_flag = word + 2;
    volatile uint32_t* const issued = word + 4;  // [stream] rounds of products issued so far
    // softmax's cells (streams 0 and 1), the cells after them, the products' (streams 0 and 1), the loads'
    Item* const items = reinterpret_cast<Item*>(tail_ptr + kItemsAt);
    float2* const exchange = reinterpret_cast<float2*>(items + kItems);  // [stream][row] (maximum, sum)

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t n_seqs = p.batch.n_seqs, group = p.group, window = p.window, cta = blockIdx.x;
    const uint32_t room = room_of(p.batch, p.pool.page_shift);

    // ---- set-up and the batch summed up --------------------------------------------------------------------------------
    if (tid == 0) {
        for (uint32_t i = 0; i < NST; ++i) {
            tc::mbar_init(bar_full + 8 * i, 1);
            tc::mbar_init(bar_empty + 8 * i, 2);  // both streams
        }
        for (uint32_t i = 0; i < 2; ++i) {
            tc::mbar_init(bar_s + 8 * i, 1);
            tc::mbar_init(bar_p + 16 * i, 128);
            tc::mbar_init(bar_p + 16 * i + 8, 128);
            tc::mbar_init(bar_o + 8 * i, 1);
            tc::mbar_init(bar_q + 8 * i, 128);
            tc::mbar_init(bar_t + 8 * i, 1);
            issued[i] = 0;
        }
        tc::mbar_init(bar_land, 1);
        tc::mbar_init(bar_done, 2);
        *abort_flag = 0;
        tc::fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        tc::tmem_alloc(smem_u32(word), kTmemCols);
        tc::tmem_relinquish();
    }
    after_predecessor();
    uint64_t* const prefix = reinterpret_cast<uint64_t*>(smem + 2 * Sh::kQ);  // [n_seqs + 1], scratch in the ring
    uint64_t* const per_head = prefix + n_seqs + 1;  // [n_seqs] tiles of one KV head
    SeqInfo* const info = reinterpret_cast<SeqInfo*>(per_head + n_seqs);
    constexpr uint64_t kLater = ~0ull;
    constexpr uint32_t kOwnBlocks = 8;  // a sequence of more blocks is summed by a whole warp
    for (uint32_t s = tid; s < n_seqs; s += kThreads) {
        Batch b = p.batch;
        if (cta != 0) b.status = nullptr;  // one CTA reports
        const Seq sq = seq_of(b, s, p.pool.page_shift);
        const SeqInfo q{sq.row0, sq.rows, sq.len};
        info[s] = q;
        const uint32_t blocks = (q.rows * group + kBlockPairs - 1) / kBlockPairs;
        uint64_t sum = kLater;
        if (blocks <= kOwnBlocks) {
            sum = 0;
            for (uint32_t i = 0; i < blocks; ++i) sum += cell_tiles(q, i, group, window, room) + kCellCost;
        }
        per_head[s] = sum;
    }
    __syncthreads();
    for (uint32_t s = warp; s < n_seqs; s += kThreads / 32) {
        if (per_head[s] != kLater) continue;
        const SeqInfo q = info[s];
        const uint32_t blocks = (q.rows * group + kBlockPairs - 1) / kBlockPairs;
        uint64_t sum = 0;
        for (uint32_t i = lane; i < blocks; i += 32) sum += cell_tiles(q, i, group, window, room) + kCellCost;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        __syncwarp();
        if (lane == 0) per_head[s] = sum;
    }
    __syncthreads();
    if (warp == 0) {  // prefix sums, 32 sequences at a time
        uint64_t base = 0;
        for (uint32_t s0 = 0; s0 < n_seqs; s0 += 32) {
            const uint32_t s = s0 + lane;
            const uint64_t mine = s < n_seqs ? per_head[s] * p.pool.kv_heads : 0u;
            uint64_t incl = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint64_t o = __shfl_up_sync(0xffffffffu, incl, d);
                if (lane >= static_cast<uint32_t>(d)) incl += o;
            }
            if (s < n_seqs) prefix[s] = base + incl - mine;
            base += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) prefix[n_seqs] = base;
    }
    __syncthreads();
    const uint64_t W = prefix[n_seqs];
    const uint64_t per = max((W + gridDim.x - 1) / gridDim.x, static_cast<uint64_t>(1));
    const uint64_t snap = min(static_cast<uint64_t>(kSnap), per / 2);
    // CTA c's run is [cut(c), cut(c + 1)): warps 0 and 1 work the two out.
    if (warp < 2) {
        uint64_t pos = (cta + warp) * per;
        uint32_t s = 0, kvh = 0, block = 0, blocks = 0;
        uint64_t left = 0;
        SeqInfo q{0, 0, 0};
        if (pos < W) {
            uint32_t lo = 0, hi = n_seqs;  // the last sequence that begins at or before pos and is not empty
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (prefix[mid] <= pos)
                    lo = mid;
                else
                    hi = mid;
            }
            s = lo;
            q = info[s];
            const uint64_t in = pos - prefix[s];
            kvh = static_cast<uint32_t>(in / per_head[s]);
            left = in % per_head[s];
            blocks = (q.rows * group + kBlockPairs - 1) / kBlockPairs;
            uint32_t tiles = 0;  // of that block
            for (uint32_t b0 = 0; b0 < blocks; b0 += 32) {  // the block that holds position `left` of the KV head
                const uint32_t mine = b0 + lane < blocks ? cell_tiles(q, b0 + lane, group, window, room) + kCellCost : 0u;
                uint32_t incl = mine;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const uint32_t o = __shfl_up_sync(0xffffffffu, incl, d);
                    if (lane >= static_cast<uint32_t>(d)) incl += o;
                }
                const uint32_t here = __ballot_sync(0xffffffffu, incl > left);
                if (here != 0u) {
                    const int at = __ffs(here) - 1;
                    block = b0 + at;
                    left -= __shfl_sync(0xffffffffu, incl - mine, at);
                    tiles = __shfl_sync(0xffffffffu, mine, at) - kCellCost;
                    break;
                }
                left -= __shfl_sync(0xffffffffu, incl, 31);
            }
            if (left <= snap) {
                pos -= left;
                left = 0;
            } else if (left + snap >= tiles) {  // to the next cell
                pos += tiles + kCellCost - left;
                left = 0;
                if (++block == blocks) {
                    block = 0;
                    if (++kvh == p.pool.kv_heads) {
                        kvh = 0;
                        do ++s;
                        while (s < n_seqs && info[s].rows == 0);
                        if (s < n_seqs) q = info[s];
                        blocks = (q.rows * group + kBlockPairs - 1) / kBlockPairs;
                    }
                }
            }
        }
        if (lane == 0) {
            Item& x = items[warp];
            x.pos = min(pos, W);
            x.s = s;
            x.kvh = kvh;
            x.block = block;
            x.blocks = blocks;
            x.off = static_cast<uint32_t>(left);
            x.q = q;
        }
    }
    __syncthreads();
    const uint64_t run0 = items[0].pos, run1 = items[1].pos;
    const bool works = run0 < run1;
    const Run run{p, run1, room};
    __syncthreads();
    if (works && warp == 0) {
        if (lane == 0) run.open_cell(items[0], items[0].off);
        __syncwarp();
        if (lane > 0 && lane < kItems) items[lane] = items[0];
    }
    tc::fence_proxy_async();  // the ring was the planning's scratch, TMA writes it next
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = word[0];
    // Waits that ran out end the call: every role leaves (or, the softmax threads, walks on through their barriers without
    // waiting), once what the role has in flight has come to rest.  A warp of the softmax that has given up is `dead`: its rows,
    // of this cell and of all that follow in the run, become NaN - by way of a maximum and sum of NaN, which every join hands
    // on - and its tickets are taken all the same, so that the workspace is as the next launch wants it.
    auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
        if (tc::mbar_try_wait(bar, parity)) return true;
        const long long t0 = clock64();
        while (!tc::mbar_try_wait(bar, parity)) {
            if (*abort_flag != 0) return false;
            if (clock64() - t0 > p.wait_clocks) {
                *abort_flag = 1;
                raise(p.batch, kWaitRanOut);
                return false;
            }
        }
        return true;
    };

    if (warp >= kMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kOtherRegs));
        if (warp == kLoadWarp && works) {
            // ---------------- loads ------------------------------------------------------------------------------------
            const uint32_t shift = p.pool.page_shift, box_shift = min(shift, 7u);  // rows of a box: a page's, or a tile's
            constexpr uint32_t NP = D / 64;
            const uint32_t slot = lane / NP, panel = lane % NP;  // lane's page within the tile, and its 64 channels
            const uint32_t row_at = slot << box_shift;           // its first row in the tile
            uint32_t cnt = 0, landed = 0;
            bool ok = true, landing = false;
            Item& it = items[6];
            do {
                const uint32_t* const tab = p.batch.table + static_cast<size_t>(it.s) * p.batch.table_stride;
                const uint32_t lo = it.lo, hi = it.hi;
                auto holds = [&](uint32_t key) { return row_at < kTile && key < hi && key + (1u << box_shift) > lo; };
                auto page_of = [&](uint32_t key) { return holds(key) ? tab[key >> shift] : 0u; };
                uint32_t ahead = it.t0 < it.t1 ? page_of(it.t0 * kTile + row_at) : 0u;  // page numbers come a tile ahead
                for (uint32_t t = it.t0; ok && t < it.t1; ++t) {
                    const uint32_t key = t * kTile + row_at;  // the box holds keys [key, key + box rows)
                    const bool mine = holds(key);
                    uint32_t page = ahead;
                    if (t + 1 < it.t1) ahead = page_of(key + kTile);
                    if (mine && page >= p.pool.n_pages) {
                        raise(p.batch, kBadPage);
                        page = p.pool.n_pages;  // outside the map: zeros
                    }
                    const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, mine));
                    const uint32_t bytes = boxes << (box_shift + 7);
                    const uint32_t a = it.lo > t * kTile ? it.lo - t * kTile : 0u, b = min(it.hi - t * kTile, kTile);
                    const bool cut = a != 0 || b != kTile;  // rows outside [a, b) are not the block's
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        const uint32_t st = cnt % NST;
                        if (cnt >= NST && !wait(bar_empty + 8 * st, (cnt / NST - 1) & 1u)) ok = false;
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        const uint32_t dst = ring + st * Sh::kStage, bar = bar_full + 8 * st;
                        const uint32_t signal = v == 1 && cut ? bar_land : bar;
                        if (lane == 0) mbar_arrive_expect(signal, bytes);
                        __syncwarp();
                        if (mine)
                            tma_load(dst + panel * Sh::kPanel + row_at * 128, v == 0 ? &kmap : &vmap, signal, panel * 64,
                                     static_cast<int32_t>(key & ((1u << shift) - 1u)), static_cast<int32_t>(it.kvh), static_cast<int32_t>(page));
                        if (v == 1 && cut) {
                            landing = true;
                            if (!wait(bar_land, landed & 1u)) ok = false;
                            ok = __all_sync(0xffffffffu, ok);
                            if (!ok) break;
                            landing = false;
                            ++landed;
                            unsigned char* const rows = smem + (dst - qbuf);
                            const uint32_t gone = kTile - (b - a);
                            for (uint32_t i = lane; i < gone * (D / 8); i += 32) {
                                const uint32_t j = i / (D / 8), c = i % (D / 8);
                                const uint32_t r = j < a ? j : b + (j - a);
                                *reinterpret_cast<uint4*>(rows + (c / 8) * Sh::kPanel + r * 128 + (c % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
                            }
                            tc::fence_proxy_async();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(bar);
                        }
                        ++cnt;
                    }
                }
                __syncwarp();
                if (lane == 0) run.next(it);
                __syncwarp();
            } while (ok && it.more);
            if (!ok) {  // copies in flight land before the block's shared memory goes
                for (uint32_t n = cnt > NST ? cnt - NST : 0u; n < cnt; ++n)
                    tc::mbar_wait_bounded(bar_full + 8 * (n % NST), (n / NST) & 1u, kRestClocks);
                if (landing) tc::mbar_wait_bounded(bar_land, landed & 1u, kRestClocks);
            }
        } else if ((warp == kMmaWarp || warp == kMmaWarp + 2) && works && lane == 0) {
            // ---------------- products of one stream ---------------------------------------------------------------------
            // A round is O += P V(t), S = Q K(t + 1).  The streams take turns round by round: left alone they fall into step,
            // both softmaxes at a time and both products at a time, each of the two waiting for the other half of the SM
            // (4400 clocks for two rounds).  One issuing thread each, since between two rounds a thread needs 500 clocks for
            // waits, releases and descriptors (with one for both the tensor core idled for 1300 of every 2400 clocks): what can
            // be waited for is waited for before the turn, and stages are released behind the round.
            const uint32_t i = (warp - kMmaWarp) / 2;
            constexpr uint32_t kType = std::is_same<P, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
            constexpr uint32_t kIdS = tc::instr_desc_f16(128, kTile, false) | kType;
            constexpr uint32_t kIdO = tc::instr_desc_f16(128, D, true) | kType;
            constexpr uint64_t kDescK = tc::smem_desc_base(16, 1024), kDescV = tc::smem_desc_base(Sh::kPanel, 1024);
            const uint32_t tS = tmem + i * kTile, tO = tmem + kTmemO + i * D;
            uint32_t base = 0, next = 0;  // the ring's count at the item's first tile; the next place to pass
            uint32_t n_p = 0, n_items = 0, mine = 0, turns = 0;  // turns: the other stream's rounds of the cells before
            auto wait_round = [&](uint32_t n) -> bool {  // until the other stream has issued its round n
                if (static_cast<int32_t>(issued[1 - i] - n) > 0) return true;
                const long long t0 = clock64();
                while (static_cast<int32_t>(issued[1 - i] - n) <= 0) {
                    if (*abort_flag != 0) return false;
                    if (clock64() - t0 > p.wait_clocks) {
                        *abort_flag = 1;
                        raise(p.batch, kWaitRanOut);
                        return false;
                    }
                }
                return true;
            };
            bool ok = true;
            Item& it = items[4 + i];
            do {
                const uint32_t t0 = it.t0, step = it.step, twin = it.twin, a = it.a[i], e = it.e[i];
                const uint64_t q = kDescK + ((qbuf + (twin != 0 ? 0u : i * Sh::kQ)) >> 4);
                // Every place of the ring goes through both threads' hands, in order: a tile that this stream does not take is
                // waited for and released too, so that no stage's barrier can run two phases ahead of a thread that tells
                // phases by their parity.
                auto reach = [&](uint32_t cn) -> bool {
                    for (; next != cn; ++next) {
                        if (!wait(bar_full + 8 * (next % NST), (next / NST) & 1u)) return false;
                        mbar_arrive(bar_empty + 8 * (next % NST));
                    }
                    return true;
                };
                auto full = [&](uint32_t cn) -> bool {
                    if (!reach(cn) || !wait(bar_full + 8 * (cn % NST), (cn / NST) & 1u)) return false;
                    ++next;
                    return true;
                };
                auto release = [&](uint32_t cn) { tc::mma_commit(bar_empty + 8 * (cn % NST)); };  // once its products are complete
                auto scores = [&](uint32_t cn) {  // S = Q K(t)
                    const uint64_t k = kDescK + ((ring + cn % NST * Sh::kStage) >> 4);
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks) {
                        if (ks == D / 32) issued[i] = ++mine;  // the other thread takes a while to see it
                        constexpr uint32_t kPanel16 = Sh::kPanel / 16;
                        const uint32_t off = (ks / 4) * kPanel16 + (ks % 4) * 2;
                        tc::mma_f16_ss(tS, q + off, k + off, kIdS, ks > 0 ? 1u : 0u);
                        if constexpr (SPLIT) tc::mma_f16_ss(tS, q + Sh::kStage / 16 + off, k + off, kIdS, 1u);
                    }
                };
                // A twin cell's queries are the first warpgroup's for both streams.  No queries are handed over before both
                // streams that read the ones before have come here (bar_t), so no phase can be passed over: stream 1 has its own
                // barrier's phase of a twin cell only after warpgroup 0 has met warpgroup 1 at the end of the cell before.
                ok = wait(bar_q + 8 * i, n_items & 1u) && (twin == 0 || i == 0 || wait(bar_q, n_items & 1u));
                if (ok) mbar_arrive(bar_t + 8 * i);
                const uint32_t xa = it.a[1 - i], xe = it.e[1 - i];
                const uint32_t rounds = xa < xe ? (xe - xa + step - 1) / step + 1 : 0u;  // of the other stream: 0, 1, ...
                // One copy of the code: the first round has no weights to use yet, the last no scores to make.
                uint32_t after = i == 0 ? 0xffffffffu : 0u;  // the other stream's round that this one follows (stream 0 begins)
                for (uint32_t nt = a; ok && a < e; nt += step, ++after) {
                    const bool have = nt != a, more = nt < e;  // weights of tile t; scores of tile nt to come
                    const uint32_t t = nt - step;
                    const uint32_t cv = base + 2 * (t - t0) + 1, ck = base + 2 * (nt - t0);
                    // (with three stages K(t + 2) takes the place of V(t), which has to be used first)
                    constexpr bool kAhead = NST >= 5;
                    if (have) ok = full(cv);
                    if (ok && more && (kAhead || twin == 0 || !have)) ok = full(ck);
                    if (ok && have) ok = wait(bar_p + 16 * i, n_p & 1u);
                    if (ok && after < rounds) ok = wait_round(turns + after);
                    if (ok && have) {  // O (+)= P V(t)
                        tc::fence_after_sync();
                        const uint64_t v = kDescV + ((ring + cv % NST * Sh::kStage) >> 4);
                        [[maybe_unused]] const uint32_t acc = t != a ? 1u : 0u;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            if (j == 4) {
                                ok = wait(bar_p + 16 * i + 8, n_p & 1u);
                                if (!ok) break;
                                tc::fence_after_sync();
                            }
                            if constexpr (SPLIT) {  // (the softmax takes every tile's output out)
                                tc::mma_f16_ts(tO, tS + 16 * j, v + j * 128, kIdO, j > 0 ? 1u : 0u);
                                tc::mma_f16_ts(tO, tS + 16 * j + 8, v + j * 128, kIdO, 1u);
                            } else {
                                tc::mma_f16_ts(tO, tS + 8 * j, v + j * 128, kIdO, j > 0 ? 1u : acc);
                            }
                        }
                        ++n_p;
                        if (!kAhead && twin != 0) {
                            release(cv);
                            if (ok && more) ok = full(ck);
                        }
                    }
                    if (!ok) break;
                    if (more) {
                        tc::fence_after_sync();
                        scores(ck);
                        tc::mma_commit(bar_s + 8 * i);
                        release(ck);
                    } else {
                        issued[i] = ++mine;
                        tc::mma_commit(bar_o + 8 * i);
                    }
                    if (have && (kAhead || twin == 0)) release(cv);
                    if (!more) break;
                }
                base += 2 * (it.t1 - t0);
                ok = ok && reach(base);
                turns += rounds;
                ++n_items;
                run.next(it);
            } while (ok && it.more);
            tc::mma_commit(bar_done);
            tc::mbar_wait_bounded(bar_done, 0u, kRestClocks);
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kSoftmaxRegs));
        // ---------------- softmax: thread r of warpgroup i owns row r of stream i ----------------------------------------
        const uint32_t i = warp >> 2, r = tid & 127;
        const uint32_t lane_base = ((warp & 3) * 32) << 16;
        const uint32_t tS = tmem + lane_base + i * kTile, tO = tmem + lane_base + kTmemO + i * D;
        const float c = fmaxf(fabsf(p.scale_log2), 1e-30f);  // the queries carry a negative scale's sign
        const bool flip = p.scale_log2 < 0.f;
        const uint32_t head_dim = p.pool.head_dim;
        uint32_t n_s = 0, n_o = 0, n_t = 0;  // scores seen, last products seen, cells ended
        bool dead = !works;         // a wait ran out: walk on through the barriers, touch nothing
        Item &it = items[i], &nx = items[2 + i];  // the warpgroup's cell and the one after it
        auto group_sync = [&]() {
            if (i == 0)
                asm volatile("bar.sync 2, 128;\n" ::: "memory");
            else
                asm volatile("bar.sync 3, 128;\n" ::: "memory");
        };
        // A row of Q, and of the output on its way out, lies in the stream's query tile: 16-byte chunk k of row x here.
        unsigned char* const qs = smem + i * Sh::kQ;
        auto chunk_at = [&](uint32_t x, uint32_t k) { return qs + (k / 8) * Sh::kPanel + x * 128 + (((k % 8) ^ (x & 7)) << 4); };
        // A block's queries into shared memory, a warp its own 32 rows, 16 bytes of channels a lane.  This, like all that runs
        // once a cell, is a rolled loop: its code is never in the instruction cache when its turn comes, and straight-line
        // code is fetched at about a byte a clock (16 unrolled loads took 5000 clocks to issue).
        constexpr uint32_t CH = D / 8, RP = 32 / CH;  // lanes of a row, rows of a pass; CH passes for a warp's 32 rows
        auto fetch_queries = [&](const Item& n) {
            const uint32_t in = i * kTile + r, pair = n.block * kBlockPairs + in;
            const bool has = in < n.pairs;
            const int64_t mine = has ? static_cast<int64_t>((n.q.row0 + pair / group) * p.q_row + (n.kvh * group + pair % group) * head_dim) : -1;
            if (i == 1 && n.twin) return;  // both streams read stream 0's
            const uint32_t ch = (lane % CH) * 8;
            const T* const q = static_cast<const T*>(p.q);
            if (SPLIT || flip) {
                constexpr uint32_t QB = 4;
#pragma unroll 1
                for (uint32_t j0 = 0; j0 < CH; j0 += QB) {
                    Vec8<T> x[QB];
#pragma unroll
                    for (uint32_t j = 0; j < QB; ++j) {
                        const int64_t off = __shfl_sync(0xffffffffu, mine, (j0 + j) * RP + lane / CH);
                        x[j] = Vec8<T>{};
                        if (off >= 0 && ch < head_dim) x[j].load(q + off + ch);
                    }
#pragma unroll
                    for (uint32_t j = 0; j < QB; ++j) {
                        unsigned char* const dst = chunk_at((warp & 3) * 32 + (j0 + j) * RP + lane / CH, lane % CH);
                        if constexpr (SPLIT) {
                            float f[8];
                            x[j].get(f);
                            uint32_t hi[4], lo[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                __half h0, l0, h1, l1;
                                split_half(flip ? -f[2 * e] : f[2 * e], h0, l0);
                                split_half(flip ? -f[2 * e + 1] : f[2 * e + 1], h1, l1);
                                hi[e] = pack_half2(h0, h1);
                                lo[e] = pack_half2(l0, l1);
                            }
                            *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                            *reinterpret_cast<uint4*>(dst + Sh::kStage) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                        } else {
                            const uint4 v = x[j].w;
                            *reinterpret_cast<uint4*>(dst) = make_uint4(v.x ^ 0x80008000u, v.y ^ 0x80008000u, v.z ^ 0x80008000u, v.w ^ 0x80008000u);
                        }
                    }
                }
            } else {
#pragma unroll 2
                for (uint32_t j = 0; j < CH; ++j) {
                    const int64_t off = __shfl_sync(0xffffffffu, mine, j * RP + lane / CH);
                    const bool live = off >= 0 && ch < head_dim;
                    cp_async16(smem_u32(chunk_at((warp & 3) * 32 + j * RP + lane / CH, lane % CH)), q + (live ? off + ch : 0), live ? 16u : 0u);
                }
            }
        };
        auto hand_over_queries = [&]() {
            asm volatile("cp.async.wait_all;\n" ::: "memory");
            tc::fence_proxy_async();
            tc::fence_before_sync();  // the next products overwrite what was read out of tensor memory
            mbar_arrive(bar_q + 8 * i);
        };
        if (works) {
            if (r == 0) run.next(nx);
            fetch_queries(it);
            hand_over_queries();
            group_sync();
        }
        while (works && it.more) {
            const uint32_t in = it.twin ? r : i * kTile + r;  // pair within the block
            const bool live = in < it.pairs;
            const uint32_t pair = it.block * kBlockPairs + (live ? in : 0u);
            const int32_t pos0 = static_cast<int32_t>(it.q.len) - static_cast<int32_t>(it.q.rows);
            const int32_t pos = live ? pos0 + static_cast<int32_t>(pair / group) : -1;
            // keys (low, at] are seen (a position may lie behind the last key)
            const int32_t low = window != 0 ? pos - static_cast<int32_t>(min(window, 0x7fffffffu)) : -1, at = min(pos, static_cast<int32_t>(room) - 1);
            float m = -INFINITY, l = 0.f;
            float acc[SPLIT ? D : 1];  // f32 rows: the output so far
#pragma unroll
            for (int u = 0; u < (SPLIT ? D : 1); ++u) acc[u] = 0.f;
            auto take_output = [&]() {
                if constexpr (SPLIT) {
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) {
                        uint32_t o[16];
                        tc::tmem_ld16(tO + 16 * j, o);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int u = 0; u < 16; ++u) acc[16 * j + u] += __uint_as_float(o[u]);
                    }
                }
            };
            auto rescale_output = [&](float f) {  // the scores at hand vouch for every product before them: O is at rest
#pragma unroll 1
                for (int j = 0; j < D; j += 16) {
                    uint32_t o[16];
                    tc::tmem_ld16(tO + j, o);
                    tc::tmem_wait_ld();
#pragma unroll
                    for (int u = 0; u < 16; ++u) o[u] = __float_as_uint(__uint_as_float(o[u]) * f);
                    tc::tmem_st16(tO + j, o);
                }
            };
            auto stored = [&](uint32_t half) {  // the weights of half of the tile's keys may be used
                tc::tmem_wait_st();
                tc::fence_before_sync();
                mbar_arrive(bar_p + 16 * i + 8 * half);
            };
            const uint32_t a = it.a[i], e = it.e[i], step = it.step;
            const bool any = a < e;
            uint32_t turn = 0;  // tiles of this cell done
            for (uint32_t t = a; t < e; t += step, ++turn) {
                dead = dead || !wait(bar_s + 8 * i, n_s & 1u);
                dead = __any_sync(0xffffffffu, dead);
                if (dead) break;
                ++n_s;
                tc::fence_after_sync();
                const int32_t from = low - static_cast<int32_t>(t * kTile), to = at - static_cast<int32_t>(t * kTile);  // columns (from, to]
                if (__any_sync(0xffffffffu, live && (from >= 0 || to < static_cast<int32_t>(kTile) - 1))) {
                    // Scores of keys that a row does not see become -infinity where they lie, in a rolled loop over the blocks
                    // that need it: few tiles do, and the loop that every tile runs through stays short.
#pragma unroll 1
                    for (int32_t col = 0; col < static_cast<int32_t>(kTile); col += 16) {
                        if (!__any_sync(0xffffffffu, live && (col <= from || col + 15 > to))) continue;
                        uint32_t x[16];
                        tc::tmem_ld16(tS + col, x);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int u = 0; u < 16; ++u)
                            if (col + u <= from || col + u > to) x[u] = 0xff800000u;
                        tc::tmem_st16(tS + col, x);
                    }
                    tc::tmem_wait_st();
                }
                if constexpr (SPLIT) {
                    // The tensor core cuts its sums short of a rounding, which adds up over a long accumulation (2.8e-6 of the
                    // norm at 2048 keys, against 0.8e-6): every tile's output is taken out of tensor memory and added here,
                    // and the scores are read twice to make room for it.
                    if (turn != 0) take_output();
                    float mx = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t x[32];
                        tc::tmem_ld32(tS + 32 * j, x);
                        tc::tmem_wait_ld();
                        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                        for (int u = 0; u < 32; u += 4) {
                            top[0] = max3(top[0], __uint_as_float(x[u]), __uint_as_float(x[u + 1]));
                            top[1] = max3(top[1], __uint_as_float(x[u + 2]), __uint_as_float(x[u + 3]));
                        }
                        mx = max3(mx, top[0], top[1]);
                    }
                    mx *= c;
                    const bool grow = mx > m + kRescaleStep || (m == -INFINITY && mx > m);
                    if (__any_sync(0xffffffffu, grow)) {
                        const float f = grow ? (m == -INFINITY ? 0.f : fast_exp2(m - mx)) : 1.f;
#pragma unroll
                        for (int u = 0; u < D; ++u) acc[u] *= f;
                        if (grow) m = mx;
                        l *= f;
                    }
                    if (!(mx < INFINITY)) m = NAN;  // a NaN or +infinity among the scores: the row is NaN from here on
                    const float nm = m == -INFINITY ? 0.f : -m;
                    // (lifted behind the exponential: 7 in its argument would cost the largest weights three of their bits)
                    const uint64_t c2 = pair_of(c, c), nm2 = pair_of(nm, nm), lift2 = pair_of(1.f / kUnlift<P>, 1.f / kUnlift<P>);
                    uint64_t sum2[2] = {0u, 0u};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t x[32];
                        tc::tmem_ld32(tS + 32 * j, x);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int g = 0; g < 2; ++g) {  // 16 keys: high terms in their columns 0-7, low terms in 8-15
                            uint32_t y[16];
#pragma unroll
                            for (int u = 0; u < 8; ++u) {
                                const float2 e2 = unpair(fma2(pair_of(__uint_as_float(x[16 * g + 2 * u]), __uint_as_float(x[16 * g + 2 * u + 1])), c2, nm2));
                                const uint64_t w2 = mul2(pair_of(fast_exp2(e2.x), fast_exp2(e2.y)), lift2);
                                sum2[u & 1] = add2(sum2[u & 1], w2);
                                const float2 w = unpair(w2);
                                const __half2 h = __floats2half2_rn(w.x, w.y);
                                const float2 hf = __half22float2(h);
                                y[u] = *reinterpret_cast<const uint32_t*>(&h);
                                y[8 + u] = pack2(__half(), w.x - hf.x, w.y - hf.y);
                            }
                            tc::tmem_st16(tS + 32 * j + 16 * g, y);
                        }
                        if (j == 1) stored(0);
                    }
                    const float2 s01 = unpair(add2(sum2[0], sum2[1]));
                    l += s01.x + s01.y;
                } else {
                    uint32_t x[4][32];
#pragma unroll
                    for (int j = 0; j < 4; ++j) tc::tmem_ld32(tS + 32 * j, x[j]);
                    tc::tmem_wait_ld();
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int u = 0; u < 32; u += 2)
#pragma unroll
                        for (int j = 0; j < 4; ++j) top[j] = max3(top[j], __uint_as_float(x[j][u]), __uint_as_float(x[j][u + 1]));
                    const float mx = max3(max3(top[0], top[1], top[2]), top[3], top[3]) * c;
                    const bool grow = mx > m + kRescaleStep || (m == -INFINITY && mx > m);
                    if (__any_sync(0xffffffffu, grow)) {
                        const float f = grow ? (m == -INFINITY ? 0.f : fast_exp2(m - mx)) : 1.f;
                        if (turn != 0) rescale_output(f);
                        if (grow) m = mx;
                        l *= f;
                    }
                    if (!(mx < INFINITY)) m = NAN;
                    const uint64_t c2 = pair_of(c, c), nm2 = pair_of(m == -INFINITY ? 0.f : kLift<P> - m, m == -INFINITY ? 0.f : kLift<P> - m);
                    uint64_t sum2[2] = {0u, 0u};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t y[16];
#pragma unroll
                        for (int u = 0; u < 16; ++u) {
                            float2 e2 = unpair(fma2(pair_of(__uint_as_float(x[j][2 * u]), __uint_as_float(x[j][2 * u + 1])), c2, nm2));
                            e2 = make_float2(fast_exp2(e2.x), fast_exp2(e2.y));
                            sum2[u & 1] = add2(sum2[u & 1], pair_of(e2.x, e2.y));
                            y[u] = pack2(P(), e2.x, e2.y);
                        }
                        tc::tmem_st16(tS + 16 * j, y);
                        if (j == 1) stored(0);
                    }
                    const float2 s01 = unpair(add2(sum2[0], sum2[1]));
                    l += s01.x + s01.y;
                }
                stored(1);
            }
            if (any && !dead) {
                dead = !wait(bar_o + 8 * i, n_o & 1u);
                dead = __any_sync(0xffffffffu, dead);
                ++n_o;
                tc::fence_after_sync();
                if constexpr (SPLIT) {  // back to where the cell's end expects it
                    if (!dead) {
#pragma unroll
                        for (int j = 0; j < D / 16; ++j) {
                            uint32_t o[16];
                            tc::tmem_ld16(tO + 16 * j, o);
                            tc::tmem_wait_ld();
#pragma unroll
                            for (int u = 0; u < 16; ++u) o[u] = __float_as_uint(acc[16 * j + u] + __uint_as_float(o[u]));
                            tc::tmem_st16(tO + 16 * j, o);
                        }
                        tc::tmem_wait_st();
                    }
                }
            }

            // ---- the cell's end ----------------------------------------------------------------------------------------
            if (dead) m = l = NAN;
            const bool whole = it.n == it.T, twin = it.twin != 0;
            float f0 = 1.f, f1 = 0.f;  // twin: weights of stream 0's and stream 1's rows
            const bool any0 = twin ? it.a[0] < it.e[0] : any, any1 = twin && it.a[1] < it.e[1];
            if (twin) {
                // Rows are the same in both streams and sit in the same lanes: each warpgroup takes half of the channels.  Both
                // add stream 0 and stream 1 in this order: the sum that one hands to a join has to be the other's, to the
                // bit, or a result's bits would depend on which CTA comes last.
                exchange[tid] = make_float2(m, l);
                tc::fence_before_sync();
                both_sync();
                tc::fence_after_sync();
                const float2 x = exchange[tid ^ 128];
                const float m0 = i == 0 ? m : x.x, m1 = i == 0 ? x.x : m, l0 = i == 0 ? l : x.y, l1 = i == 0 ? x.y : l;
                const float M = m0 != m0 || m1 != m1 ? NAN : fmaxf(m0, m1);
                f0 = m0 == -INFINITY ? 0.f : fast_exp2(m0 - M);
                f1 = m1 == -INFINITY ? 0.f : fast_exp2(m1 - M);
                l = fmaf(l0, f0, l1 * f1);
                m = M;
            }
            const uint32_t row = it.q.row0 + pair / group, head = it.kvh * group + pair % group;
            const uint32_t c0 = twin ? i * (D / 2) : 0u, c1 = twin ? c0 + D / 2 : D;  // channels of this thread
            const int64_t dst = live ? static_cast<int64_t>(row * p.out_row + head * head_dim) : -1;
            const uint32_t tO0 = twin ? tmem + lane_base + kTmemO : tO, tO1 = tmem + lane_base + kTmemO + D;
            auto output16 = [&](uint32_t ch, float (&f)[16]) {
                uint32_t o[16] = {}, y[16] = {};
                if (!dead) {
                    tc::tmem_ld16(tO0 + ch, o);
                    if (twin) tc::tmem_ld16(tO1 + ch, y);
                    tc::tmem_wait_ld();
                }
#pragma unroll
                for (int u = 0; u < 16; ++u) {
                    f[u] = any0 ? __uint_as_float(o[u]) : 0.f;
                    if (twin) f[u] = fmaf(f[u], f0, any1 ? __uint_as_float(y[u]) * f1 : 0.f);
                }
            };
            // A finished row goes out by way of shared memory, so that a warp stores whole rows: thread by thread, 32 rows at
            // a time, every store would touch 32 lines (7000 clocks a cell).
            auto stage16 = [&](uint32_t ch, const float (&f)[16], float by) {
                if constexpr (SPLIT) {
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        *reinterpret_cast<float4*>(chunk_at(r, ch / 4 + g)) = make_float4(f[4 * g] * by, f[4 * g + 1] * by, f[4 * g + 2] * by, f[4 * g + 3] * by);
                } else {
#pragma unroll
                    for (int g = 0; g < 2; ++g)
                        *reinterpret_cast<uint4*>(chunk_at(r, ch / 8 + g)) =
                            make_uint4(pack2(P(), f[8 * g] * by, f[8 * g + 1] * by), pack2(P(), f[8 * g + 2] * by, f[8 * g + 3] * by),
                                       pack2(P(), f[8 * g + 4] * by, f[8 * g + 5] * by), pack2(P(), f[8 * g + 6] * by, f[8 * g + 7] * by));
                }
            };
            auto send_rows = [&]() {
                __syncwarp();
                constexpr uint32_t E = 16 / sizeof(T);  // channels of a chunk
                const uint32_t wide = (c1 - c0) / E, first = c0 / E;  // chunks of a row: a power of two up to 32
                const uint32_t k = first + lane % wide, sub = lane / wide, rows = 32 / wide;
#pragma unroll 4
                for (uint32_t x = 0; x < 32; x += rows) {
                    const int64_t off = __shfl_sync(0xffffffffu, dst, x + sub);
                    if (off >= 0 && k * E < head_dim)
                        *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + off + k * E) = *reinterpret_cast<const uint4*>(chunk_at((warp & 3) * 32 + x + sub, k));
                }
                __syncwarp();
            };
            auto put_lse = [&](uint32_t lrow, uint32_t lhead, float top, float sum) {
                if (p.lse)
                    p.lse[static_cast<uint64_t>(lrow) * p.q_heads + lhead] =
                        sum > 0.f || sum != sum ? (top + log2f(sum * kUnlift<P>)) * 0.69314718055994530942f : -INFINITY;
            };
            auto inverse = [](float sum) { return sum > 0.f || sum != sum ? 1.f / sum : 0.f; };
            if (whole) {
                const float inv = inverse(l);
#pragma unroll 1
                for (uint32_t ch = c0; ch < c1; ch += 16) {
                    float f[16];
                    output16(ch, f);
                    stage16(ch, f, inv);
                }
                send_rows();
                if (live && (i == 0 || !twin)) put_lse(row, head, m, l);
            } else {
                // The part goes out channels by rows: a warp's store is 512 contiguous bytes.
                const uint32_t part = it.off == 0 ? 2 * cta + 1 : 2 * cta;
                float4* const all = reinterpret_cast<float4*>(p.part_o);
                float2* const pml = reinterpret_cast<float2*>(p.part_ml);
                {
#pragma unroll 1
                    for (uint32_t ch = c0; ch < c1; ch += 16) {
                        float f[16];
                        output16(ch, f);
                        if (live) {
#pragma unroll
                            for (int g = 0; g < 4; ++g)
                                all[(static_cast<size_t>(part) * (D / 4) + ch / 4 + g) * kBlockPairs + in] = make_float4(f[4 * g], f[4 * g + 1], f[4 * g + 2], f[4 * g + 3]);
                        }
                    }
                }
                if (live && (i == 0 || !twin)) pml[static_cast<size_t>(part) * kBlockPairs + in] = make_float2(m, l);
                // The CTAs that share it: those whose runs begin inside it, and the one in whose run it begins.
                const uint64_t cell0 = it.pos - it.off;
                uint32_t first = static_cast<uint32_t>(cell0 / per), last = static_cast<uint32_t>((cell0 + it.T - 1) / per);
                if ((first + 1) * per - cell0 <= snap) ++first;  // that cut has moved to the cell's beginning
                if (last > first && last * per - cell0 + snap >= it.T) --last;  // ... and that one behind its end
                both_sync();
                if (tid == 0) {
                    const uint32_t ticket = take_ticket(p.tickets + first);
                    word[1] = ticket == last - first ? 1u : 0u;
                    if (ticket == last - first) p.tickets[first] = 0u;  // as the next launch wants it
                }
                both_sync();
                // The parts lie in slots 2 first + 1 (where the cell begins), 2 (first + 1), 2 (first + 2), ...
                const uint32_t n_parts = last - first + 1;
                auto slot_of = [&](uint32_t k) { return static_cast<size_t>(2 * (first + k) + (k == 0 ? 1 : 0)); };
                if (word[1] != 0u) {
                    if (n_parts == 2) {
                        // Every thread joins its own row, its own part still in tensor memory - in the order of the parts,
                        // whichever of the two came last, so that the same call gives the same bits.
                        const bool own_first = cta == first;
                        const size_t slot = slot_of(own_first ? 1 : 0);
                        float2 x1 = make_float2(-INFINITY, 0.f);
                        if (live) x1 = __ldcg(pml + slot * kBlockPairs + in);
                        const float M = m != m || x1.x != x1.x ? NAN : fmaxf(m, x1.x);
                        const float g0 = m == -INFINITY ? 0.f : fast_exp2(m - M), g1 = x1.x == -INFINITY ? 0.f : fast_exp2(x1.x - M);
                        const float wa = own_first ? g0 : g1, wb = own_first ? g1 : g0;
                        auto joined = [&](float own, float other) {
                            return fmaf(own_first ? other : own, wb, (own_first ? own : other) * wa);
                        };
                        const float L = joined(l, x1.y), inv = inverse(L);
                        const float4* const o1 = all + slot * (D / 4) * kBlockPairs + in;
#pragma unroll 2
                        for (uint32_t ch = c0; ch < c1; ch += 16) {
                            float f[16];
                            float4 y1[4];
#pragma unroll
                            for (int g = 0; g < 4; ++g) {
                                y1[g] = make_float4(0.f, 0.f, 0.f, 0.f);
                                if (live) y1[g] = __ldcg(o1 + static_cast<size_t>(ch / 4 + g) * kBlockPairs);
                            }
                            output16(ch, f);
#pragma unroll
                            for (int g = 0; g < 4; ++g) {
                                f[4 * g] = joined(f[4 * g], y1[g].x);
                                f[4 * g + 1] = joined(f[4 * g + 1], y1[g].y);
                                f[4 * g + 2] = joined(f[4 * g + 2], y1[g].z);
                                f[4 * g + 3] = joined(f[4 * g + 3], y1[g].w);
                            }
                            stage16(ch, f, inv);
                        }
                        send_rows();
                        if (live && (i == 0 || !twin)) put_lse(row, head, M, L);
                    } else {
                        // Threads take (row, eight channels), two such at a time and several parts of each: what a join costs
                        // is the latency of its loads.
                        constexpr uint32_t B = 5;
                        const uint32_t across = (it.pairs + 31) / 32 * 32, units = across * (head_dim / 8);
#pragma unroll 1
                        for (uint32_t u0 = tid; u0 < units; u0 += 512) {
                            float M[2] = {-INFINITY, -INFINITY}, L[2] = {}, z[2][8] = {};
                            uint32_t jr[2], c8[2];
                            bool has[2];
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t u = u0 + 256 * h;
                                jr[h] = u % across;
                                c8[h] = u / across;
                                has[h] = u < units && jr[h] < it.pairs;
                            }
#pragma unroll 1
                            for (uint32_t k0 = 0; k0 < n_parts; k0 += B) {
                                float2 ml[2][B];
                                float4 o0[2][B], o1[2][B];
#pragma unroll
                                for (int h = 0; h < 2; ++h)
#pragma unroll
                                    for (uint32_t k = 0; k < B; ++k) {
                                        const size_t sl = slot_of(min(k0 + k, n_parts - 1));
                                        ml[h][k] = make_float2(-INFINITY, 0.f);
                                        o0[h][k] = o1[h][k] = make_float4(0.f, 0.f, 0.f, 0.f);
                                        if (has[h]) {
                                            ml[h][k] = __ldcg(pml + sl * kBlockPairs + jr[h]);
                                            o0[h][k] = __ldcg(all + (sl * (D / 4) + 2 * c8[h]) * kBlockPairs + jr[h]);
                                            o1[h][k] = __ldcg(all + (sl * (D / 4) + 2 * c8[h] + 1) * kBlockPairs + jr[h]);
                                        }
                                    }
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    float to = M[h];
#pragma unroll
                                    for (uint32_t k = 0; k < B; ++k) to = max3(to, ml[h][k].x, ml[h][k].x);
                                    const float g0 = M[h] == -INFINITY ? 0.f : fast_exp2(M[h] - to);
                                    L[h] *= g0;
#pragma unroll
                                    for (int q = 0; q < 8; ++q) z[h][q] *= g0;
                                    M[h] = to;
#pragma unroll
                                    for (uint32_t k = 0; k < B; ++k) {
                                        const float g1 = k0 + k < n_parts && ml[h][k].x != -INFINITY ? fast_exp2(ml[h][k].x - to) : 0.f;
                                        L[h] += g1 * ml[h][k].y;
                                        const float4 x0 = o0[h][k], x1 = o1[h][k];
                                        z[h][0] += g1 * x0.x, z[h][1] += g1 * x0.y, z[h][2] += g1 * x0.z, z[h][3] += g1 * x0.w;
                                        z[h][4] += g1 * x1.x, z[h][5] += g1 * x1.y, z[h][6] += g1 * x1.z, z[h][7] += g1 * x1.w;
                                    }
                                }
                            }
#pragma unroll 1
                            for (int h = 0; h < 2; ++h) {
                                if (!(h == 0 ? has[0] : has[1])) continue;
                                const uint32_t row_in = h == 0 ? jr[0] : jr[1], ch = 8 * (h == 0 ? c8[0] : c8[1]);
                                const float top = h == 0 ? M[0] : M[1], sum = h == 0 ? L[0] : L[1], inv = inverse(sum);
                                float f[8];
#pragma unroll
                                for (int q = 0; q < 8; ++q) f[q] = (h == 0 ? z[0][q] : z[1][q]) * inv;
                                const uint32_t jp = it.block * kBlockPairs + row_in, jrow = it.q.row0 + jp / group, jhead = it.kvh * group + jp % group;
                                Vec8<T> v;
                                if constexpr (SPLIT) {
                                    v.set(f);
                                } else {
                                    v.w = make_uint4(pack2(P(), f[0], f[1]), pack2(P(), f[2], f[3]), pack2(P(), f[4], f[5]), pack2(P(), f[6], f[7]));
                                }
                                v.store(static_cast<T*>(p.out) + static_cast<uint64_t>(jrow) * p.out_row + jhead * head_dim + ch);
                                if (ch == 0) put_lse(jrow, jhead, top, sum);
                            }
                        }
                    }
                }
            }
            // A stream without a tile in the cell has waited for nothing of its products' thread so far: queries handed over
            // two cells ahead of it would complete a phase that it tells by its parity.
            dead = dead || !wait(bar_t + 8 * i, n_t & 1u);
            dead = __any_sync(0xffffffffu, dead);
            ++n_t;
            if (twin) {  // the other stream's accumulator and the exchange are done with
                tc::fence_before_sync();
                both_sync();
                tc::fence_after_sync();
            }
            const bool more = nx.more != 0;
            if (more) {
                // A twin cell's stream 1 reads the queries of stream 0: neither is handed over before both are free.
                if (nx.twin) both_sync();
                fetch_queries(nx);
            }
            group_sync();
            if (r == 0) {
                it = nx;
                if (more) run.next(nx);
            }
            if (more) hand_over_queries();
            group_sync();
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, kTmemCols);
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return fn;
}

// [page][head][row][channel] of a pool, boxes of 64 channels and the rows that one page has in a tile.
bool make_map(CUtensorMap* map, const Pool& pool, void* data, int32_t dtype) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) return false;
    const uint64_t rows = 1ull << pool.page_shift;
    const cuuint64_t dims[4] = {pool.head_dim, rows, pool.kv_heads, pool.n_pages};
    // (a stride of a dimension of one element is never used, and may not be zero)
    const cuuint64_t strides[3] = {rows > 1 ? pool.row_stride * 2 : 16, pool.kv_heads > 1 ? pool.head_stride * 2 : 16,
                                   pool.n_pages > 1 ? pool.page_stride * 2 : 16};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(rows < kTile ? rows : kTile), 1, 1}, one[4] = {1, 1, 1, 1};
    return encode(map, dtype == ITK_ROW_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, data, dims, strides, box,
                  one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
cudaError_t launch_as(const AttnParams& p, int32_t page_dtype, uint32_t sms, cudaStream_t s) {
    auto kernel = paged_tc_kernel<T, D>;
    static OncePerDevice prepared;
    if (!prepared.done(p.device)) {
        cudaFuncAttributes attr;
        cudaError_t e = handled(cudaFuncGetAttributes(&attr, kernel));
        if (e != cudaSuccess) return e;
        // The warpgroups' shares are drawn from what the block was launched with: fewer, and setmaxnreg would wait for good.
        if (attr.numRegs != kLaunchRegs) return cudaErrorInvalidKernelImage;
        e = handled(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Shape<T, D>::kSmem)));
        if (e != cudaSuccess) return e;
        prepared.mark(p.device);
    }
    CUtensorMap km, vm;
    if (!make_map(&km, p.pool, p.pool.k, page_dtype) || !make_map(&vm, p.pool, p.pool.v, page_dtype)) return cudaErrorInvalidValue;
    return launch_dependent(kernel, sms, kThreads, Shape<T, D>::kSmem, s, p, km, vm);
}

}  // namespace

bool tc_takes(const Pool& pool) { return pool.head_dim <= 128 && pool.page_shift >= 3; }

cudaError_t launch_tc(const AttnParams& p, int32_t row_dtype, uint32_t sms, cudaStream_t s) {
    const bool narrow = p.pool.head_dim <= 64;
    if (row_dtype == ITK_ROW_F32) return narrow ? launch_as<float, 64>(p, ITK_ROW_F16, sms, s) : launch_as<float, 128>(p, ITK_ROW_F16, sms, s);
    if (row_dtype == ITK_ROW_F16) return narrow ? launch_as<__half, 64>(p, ITK_ROW_F16, sms, s) : launch_as<__half, 128>(p, ITK_ROW_F16, sms, s);
    return narrow ? launch_as<__nv_bfloat16, 64>(p, ITK_ROW_BF16, sms, s) : launch_as<__nv_bfloat16, 128>(p, ITK_ROW_BF16, sms, s);
}

}  // namespace paged
}  // namespace itk
