// Attention of a ragged batch over the pages of its sequences, for calls with few (row, head) pairs per KV head: decode
// steps and short verify blocks - and, at any cost in speed, every shape the tensor-memory kernel does not take.
//
// For one row at position p and one head:  out = sum_k w_k v_k / sum_k w_k,  w_k = 2^(c q.k - m) (times a constant, see kLift),  c = scale * log2(e),
// over the keys p - window < k <= p, with the running maximum m and the sums kept in f32 in one pass over the keys.
//
// Bound: HBM.  Every K and V row of a (sequence, KV head) is read once for all the pairs of the KV head's group (up to
// 16), which makes 16 multiply-adds per byte at most: the mma.sync path is enough, and its 16-row operand is filled
// where a 128-row tile would be padding.
//
//   work    The launch's 64-key tiles, laid end to end over all cells (sequence, KV head, block of pairs), are cut into
//           equal runs, one per persistent CTA, from lengths that only the device knows: every CTA sums up the batch by
//           itself.  A cell that several CTAs share leaves one partial (maximum, sum, output) per CTA; the CTA that
//           takes the cell's last ticket joins them.  No CTA waits for another.
//   tiles   A warp owns 16 keys of every tile with a cp.async ring of its own, so that no barrier stands between tiles;
//           page numbers are fetched one tile ahead of the copies that need them.  Rows outside the block's keys are
//           never read: their shared-memory rows are zeros and their scores -infinity, whatever the page holds there.
//   pairs   16-bit rows: the 16 rows of a score product are 16 pairs, products exact, weights rounded to the pages'
//           type (half a step of the output's own type, and averaged over the keys).  f32 rows: x = h + l with two
//           halfs, so that 8 pairs take the 16 rows and scores and outputs come out f32-grade.
//
// Measured (us, share of the copy rate): one layer of 8 x 32768 keys, 64 / 8 heads of 128, f32 rows: 167-177 (0.94-1.0); 16 sequences
// of 256-8192 keys, bf16: 52 (0.82: 4.3 us until the first tile is there, 5-8 us of cell ends behind the stream); one sequence of
// 4096 keys: 11.4, a chain of dependent steps (lengths, page numbers, keys, the warps' exchange, ticket, join).
#include <type_traits>

#include "attn_common.cuh"
#include "paged.cuh"

namespace itk {
namespace paged {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr uint32_t kTile = 64;   // keys of a tile, 16 per warp
constexpr uint32_t kMinRun = 2;  // tiles a CTA takes at least
constexpr float kRescaleStep = 8.f;  // log2 of the growth of a maximum that triggers a rescale
// What a cell's end costs its CTA (the warps' exchange, the part's stores, its ticket: 3 us, against 1.5 us a tile), in tiles: each cell reserves
// as many beyond its own, so that runs with many ends get fewer tiles.
constexpr uint32_t kCellCost = 3;

template <typename T>
struct RowTraits;  // kPairs: (row, head) pairs that fill the 16 rows of a score product
template <>
struct RowTraits<float> {
    using Page = __half;
    static constexpr uint32_t kPairs = 8;
};
template <>
struct RowTraits<__half> {
    using Page = __half;
    static constexpr uint32_t kPairs = 16;
};
template <>
struct RowTraits<__nv_bfloat16> {
    using Page = __nv_bfloat16;
    static constexpr uint32_t kPairs = 16;
};

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename P>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<P, __half>::value)
        mma_16816(c, a, b0, b1);
    else
        mma_bf16(c, a, b0, b1);
}
__device__ __forceinline__ uint32_t pack2(__half, float x, float y) { return pack_half2(__float2half_rn(x), __float2half_rn(y)); }
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16, float x, float y) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// A sequence as the walk over the batch sees it.
struct SeqInfo {
    uint32_t row0, rows, len;  // len: as stated; there are min(len, room) keys
};

// Where a walk over a CTA's run stands: a cell and, inside it, the 64-key tiles [t, t_end) that are left to do.
struct Cursor {
    uint64_t pos, next;    // run position of the cell's first tile here, and of what follows it
    uint32_t s, kvh, b;    // sequence, KV head, block of pairs
    uint32_t blocks, T;    // of the sequence: blocks of pairs, tiles of each cell (it reserves T + kCellCost)
    uint32_t tile0;        // tile the run enters the cell at
    uint32_t row0, rows, len;
    uint32_t t, t_end;
    uint32_t lo, hi;  // keys any row of the block sees
    bool fresh, done;
};

// Shared memory grows by 20 bytes a sequence: of 128 channels, two CTAs have room on a multiprocessor up to 842 sequences (433
// with two products), one beyond - right all the same, since no CTA waits for another.
template <int D, int STAGES>
__host__ __device__ constexpr size_t pipe_bytes() {
    return static_cast<size_t>(STAGES) * kWarps * 2 * 16 * D * 2;
}
template <int D, int STAGES>
size_t smem_bytes(int mt, uint32_t n_seqs) {
    return pipe_bytes<D, STAGES>() + (mt > 1 ? mt * 16 * D * 2 : 0) + 2 * kWarps * 16 * sizeof(float) + 32 + (n_seqs + 1) * sizeof(uint64_t) +
           n_seqs * sizeof(SeqInfo);
}

// MT: score products of 16 rows a block takes.  With one, the queries stay in registers; with two they are read from shared
// memory for every tile, next to the keys they meet.
template <typename T, int D, int STAGES, int MT>
__global__ void __launch_bounds__(kThreads, D <= 128 ? 2 : 1) paged_stream_kernel(const __grid_constant__ AttnParams p) {
    using P = typename RowTraits<T>::Page;
    constexpr uint32_t PT = RowTraits<T>::kPairs, PB = MT * PT;
    constexpr bool SPLIT = PT == 8;  // two-term f32 rows
    constexpr int J = SPLIT ? 1 : 2;  // rows g, g + 8 of a product that are pairs of their own
    constexpr uint32_t kRowBytes = D * 2, kSlice = 16 * kRowBytes;
    constexpr uint32_t CH = D / 8;            // 16-byte chunks of a row
    constexpr uint32_t kPassRows = 32 / CH;   // rows a warp copies at a time
    constexpr uint32_t kPasses = 16 / kPassRows;
    constexpr int KS = D / 16, NT = D / 8;

    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char* const qs = smem + pipe_bytes<D, STAGES>();  // [MT][16][D] queries, when MT > 1
    float* wm = reinterpret_cast<float*>(qs + (MT > 1 ? MT * 16 * kRowBytes : 0));  // [warp][16]
    float* wl = wm + kWarps * 16;
    uint32_t* s_flag = reinterpret_cast<uint32_t*>(wl + kWarps * 16);
    uint64_t* s_warp = reinterpret_cast<uint64_t*>(s_flag + 8);
    uint64_t* prefix = s_warp;  // [n_seqs + 1]; its head doubles as the scan's scratch before it is filled
    SeqInfo* info = reinterpret_cast<SeqInfo*>(prefix + p.batch.n_seqs + 1);

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tq = lane & 3;
    const uint32_t n_seqs = p.batch.n_seqs, G = gridDim.x, cta = blockIdx.x;
    const uint32_t group = p.group, head_dim = p.pool.head_dim, shift = p.pool.page_shift;
    const uint32_t room = room_of(p.batch, shift);

    after_predecessor();

    // ---- the batch summed up: prefix[s] = tiles reserved before sequence s -----------------------------------------
    // A cell's block of pairs reserves the tiles of its whole sequence (of its first row's window to its last key);
    // tiles that the block does not see are passed over in the walk.
    auto geometry = [&](uint32_t rows, uint32_t len, uint32_t& lo_t, uint32_t& tiles, uint32_t& blocks) {
        const int32_t pos0 = static_cast<int32_t>(len) - static_cast<int32_t>(rows);
        lo_t = p.window != 0 && pos0 >= 0 && static_cast<uint32_t>(pos0) >= p.window ? (pos0 + 1 - p.window) / kTile : 0u;
        const uint32_t hi_t = (min(len, room) + kTile - 1) / kTile;
        tiles = hi_t > lo_t ? hi_t - lo_t : 1u;
        blocks = (rows * group + PB - 1) / PB;
    };
    const uint32_t each = (n_seqs + kThreads - 1) / kThreads;
    uint64_t mine = 0;
    for (uint32_t i = 0; i < each; ++i) {
        const uint32_t s = tid * each + i;
        if (s >= n_seqs) break;
        Batch b = p.batch;
        if (cta != 0) b.status = nullptr;  // one CTA reports
        const Seq q = seq_of(b, s, shift);
        info[s] = SeqInfo{q.row0, q.rows, q.len};
        uint32_t lo_t, tiles, blocks;
        geometry(q.rows, q.len, lo_t, tiles, blocks);
        mine += static_cast<uint64_t>(tiles + kCellCost) * blocks * p.pool.kv_heads;
    }
    uint64_t incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint64_t o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= static_cast<uint32_t>(d)) incl += o;
    }
    uint64_t* const wsum = reinterpret_cast<uint64_t*>(wm);  // [4], before the walk needs it
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    uint64_t before = incl - mine, W = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
        if (w < warp) before += wsum[w];
        W += wsum[w];
    }
    for (uint32_t i = 0; i < each; ++i) {
        const uint32_t s = tid * each + i;
        if (s >= n_seqs) break;
        prefix[s] = before;
        uint32_t lo_t, tiles, blocks;
        geometry(info[s].rows, info[s].len, lo_t, tiles, blocks);
        before += static_cast<uint64_t>(tiles + kCellCost) * blocks * p.pool.kv_heads;
    }
    if (tid == 0) prefix[n_seqs] = W;
    __syncthreads();
    uint64_t per = (W + G - 1) / G;
    if (per < kMinRun) per = kMinRun;
    const uint64_t run0 = cta * per, run1 = min(W, run0 + per);
    if (run0 >= run1) return;

    // ---- the walk ----------------------------------------------------------------------------------------------------
    auto open_seq = [&](Cursor& c) {
        const SeqInfo q = info[c.s];
        c.row0 = q.row0;
        c.rows = q.rows;
        c.len = q.len;
        uint32_t lo_t;
        geometry(q.rows, q.len, lo_t, c.T, c.blocks);
    };
    auto open_cell = [&](Cursor& c, uint32_t tile) {  // entered at reserved tile `tile`
        uint32_t lo_t, tiles, blocks;
        geometry(c.rows, c.len, lo_t, tiles, blocks);
        const uint32_t n = static_cast<uint32_t>(min(run1 - c.pos, static_cast<uint64_t>(c.T + kCellCost - tile)));
        c.next = c.pos + n;
        c.tile0 = tile;
        const uint32_t r0 = c.b * PB / group, r1 = (min(c.rows * group, (c.b + 1) * PB) - 1) / group;
        const int32_t pos0 = static_cast<int32_t>(c.len) - static_cast<int32_t>(c.rows);
        const int32_t first = pos0 + static_cast<int32_t>(r0), last = pos0 + static_cast<int32_t>(r1);
        c.hi = last >= 0 ? min(static_cast<uint32_t>(last) + 1u, room) : 0u;
        c.lo = p.window != 0 && first >= 0 && static_cast<uint32_t>(first) >= p.window ? first + 1 - p.window : 0u;
        c.t = max(lo_t + tile, c.lo / kTile);
        c.t_end = min(lo_t + min(tile + n, c.T), (c.hi + kTile - 1) / kTile);
        if (c.t >= c.t_end || c.lo >= c.hi) {  // nothing to see here: one empty step, so that the cell is still finished
            c.t = 0;
            c.t_end = 1;
            c.lo = c.hi = 0;
        }
        c.fresh = true;
    };
    auto next_cell = [&](Cursor& c) {
        c.pos = c.next;
        if (c.pos >= run1) {
            c.done = true;
            return;
        }
        if (c.pos >= prefix[c.s + 1]) {
            do ++c.s;
            while (c.pos >= prefix[c.s + 1]);
            c.kvh = c.b = 0;
            open_seq(c);
        } else if (++c.b == c.blocks) {
            c.b = 0;
            ++c.kvh;
        }
        open_cell(c, 0);
    };
    auto step = [&](Cursor& c) {
        c.fresh = false;
        if (++c.t == c.t_end) next_cell(c);
    };
    Cursor C;
    {
        uint32_t lo = 0, hi = n_seqs;  // the last sequence that begins at or before run0 and is not empty
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (prefix[mid] <= run0)
                lo = mid;
            else
                hi = mid;
        }
        C.s = lo;
        C.pos = run0;
        C.done = false;
        open_seq(C);
        const uint64_t in = run0 - prefix[lo];
        const uint32_t reserved = C.T + kCellCost;
        uint32_t cell, tile;
        if (in >> 32 == 0) {  // (a 64-bit division takes a fifth of a microsecond)
            cell = static_cast<uint32_t>(in) / reserved;
            tile = static_cast<uint32_t>(in) % reserved;
        } else {
            cell = static_cast<uint32_t>(in / reserved);
            tile = static_cast<uint32_t>(in % reserved);
        }
        C.kvh = cell / C.blocks;
        C.b = cell % C.blocks;
        if (tile >= C.T) {  // the run begins behind the cell's tiles: with the next cell
            C.next = run0 + (reserved - tile);
            next_cell(C);
            if (C.done) return;
        } else {
            open_cell(C, tile);
        }
    }
    Cursor L = C;  // the copies' walk, STAGES - 1 tiles ahead

    // ---- copies ------------------------------------------------------------------------------------------------------
    const uint32_t pipe = smem_u32(smem) + warp * (STAGES * 2 * kSlice);
    const uint32_t chunk = lane % CH, prow = lane / CH;
    const bool live_chunk = chunk * 8 < head_dim;
    const P* const kc = static_cast<const P*>(p.pool.k) + chunk * 8;
    const P* const vc = static_cast<const P*>(p.pool.v) + chunk * 8;
    const uint32_t row_mask = (1u << shift) - 1u;
    // The number of the page that holds row (lane % 16) of the slice at L, one step ahead of its use.
    auto page_of = [&]() -> uint32_t {
        const uint32_t key = L.t * kTile + warp * 16 + (lane & 15);
        const uint32_t inside = min(max(key, L.lo), L.hi - 1u);  // rows outside the block's keys are not read
        if (L.done || L.hi == 0) return 0u;
        return p.batch.table[static_cast<size_t>(L.s) * p.batch.table_stride + (inside >> shift)];
    };
    uint32_t page = page_of();
    auto request = [&](uint32_t stage) {
        const uint32_t key0 = L.t * kTile + warp * 16;
        const uint32_t a = L.lo > key0 ? min(L.lo - key0, 16u) : 0u, b = L.hi > key0 ? min(L.hi - key0, 16u) : 0u;
        if (a < b) {  // rows [a, b) of the slice are read, the others become zeros
            const bool bad = page >= p.pool.n_pages;
            if (bad) raise(p.batch, kBadPage);
            const uint32_t ks = pipe + stage * (2 * kSlice), vs = ks + kSlice;
            const uint64_t head = static_cast<uint64_t>(L.kvh) * p.pool.head_stride;
            if (shift >= 4) {  // a slice lies in one page
                const uint64_t base = bad ? 0u : page * p.pool.page_stride + (key0 & row_mask) * p.pool.row_stride + head;
                const uint64_t jump = bad ? 0u : p.pool.row_stride;
#pragma unroll
                for (uint32_t i = 0; i < kPasses; ++i) {
                    const uint32_t r = prow + i * kPassRows;
                    const uint32_t n = live_chunk && !bad && r >= a && r < b ? 16u : 0u;
                    const uint64_t off = n ? base + r * jump : 0u;
                    const uint32_t so = r * kRowBytes + ((chunk ^ (r & 7)) << 4);
                    cp_async16(ks + so, kc + off, n);
                    cp_async16(vs + so, vc + off, n);
                }
            } else {
#pragma unroll
                for (uint32_t i = 0; i < kPasses; ++i) {
                    const uint32_t r = prow + i * kPassRows;
                    const uint32_t pg = __shfl_sync(0xffffffffu, page, r);
                    const uint32_t n = live_chunk && pg < p.pool.n_pages && r >= a && r < b ? 16u : 0u;
                    const uint64_t off = n ? pg * p.pool.page_stride + ((key0 + r) & row_mask) * p.pool.row_stride + head : 0u;
                    const uint32_t so = r * kRowBytes + ((chunk ^ (r & 7)) << 4);
                    cp_async16(ks + so, kc + off, n);
                    cp_async16(vs + so, vc + off, n);
                }
            }
        }
        step(L);
        page = page_of();
    };
#pragma unroll
    for (uint32_t i = 0; i < STAGES - 1; ++i) {
        if (!L.done) request(i);
        cp_async_commit();
    }

    // ---- the pass over the run -----------------------------------------------------------------------------------------
    uint32_t qf[MT == 1 ? KS : 1][4];
    float o[MT][NT][4];
    float m[MT][J], l[MT][J];  // per product: rows g and g + 8 (f32 rows: row g alone)
    int32_t at[MT][J];         // their positions; below zero: sees nothing
    uint32_t stage = 0;
    while (!C.done) {
        const int32_t pos0 = static_cast<int32_t>(C.len) - static_cast<int32_t>(C.rows);
        if (C.fresh) {
            const uint32_t pairs = C.rows * group;
            auto query = [&](uint32_t pair) -> const T* {  // its row of Q, if there is one
                if (pair >= pairs) return nullptr;
                return static_cast<const T*>(p.q) + static_cast<uint64_t>(C.row0 + pair / group) * p.q_row + (C.kvh * group + pair % group) * head_dim;
            };
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const uint32_t pair = C.b * PB + t * PT + g + 8 * j;
                    at[t][j] = pair < pairs ? pos0 + static_cast<int32_t>(pair / group) : -1;
                    m[t][j] = -INFINITY;
                    l[t][j] = 0.f;
                }
            if constexpr (MT == 1) {
                const T* qp[2] = {query(C.b * PB + g), SPLIT ? nullptr : query(C.b * PB + g + 8)};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {  // channels 16 ks + 8 e + 2 tq and the next
                        const uint32_t d = 16 * ks + 8 * e + 2 * tq;
                        if constexpr (SPLIT) {
                            float2 x = make_float2(0.f, 0.f);
                            if (qp[0] && d < head_dim) x = *reinterpret_cast<const float2*>(qp[0] + d);
                            __half h0, l0, h1, l1;
                            split_half(x.x, h0, l0);
                            split_half(x.y, h1, l1);
                            qf[ks][2 * e] = pack_half2(h0, h1);
                            qf[ks][2 * e + 1] = pack_half2(l0, l1);
                        } else {
#pragma unroll
                            for (int j = 0; j < 2; ++j)
                                qf[ks][2 * e + j] = qp[j] && d < head_dim ? *reinterpret_cast<const uint32_t*>(qp[j] + d) : 0u;
                        }
                    }
                }
            } else {
                // Every warp has left the cell before (it ended with a barrier).  Row x of product t at [t][x].
                for (uint32_t u = tid; u < PB * CH; u += kThreads) {
                    const uint32_t pair = u / CH, ch = u % CH, t = pair / PT, x = pair % PT;
                    const T* src = query(C.b * PB + pair);
                    Vec8<T> v = {};
                    if (src && ch * 8 < head_dim) v.load(src + ch * 8);
                    unsigned char* const dst = qs + t * 16 * kRowBytes;
                    if constexpr (SPLIT) {
                        float f[8];
                        v.get(f);
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            __half h0, l0, h1, l1;
                            split_half(f[2 * e], h0, l0);
                            split_half(f[2 * e + 1], h1, l1);
                            hi[e] = pack_half2(h0, h1);
                            lo[e] = pack_half2(l0, l1);
                        }
                        *reinterpret_cast<uint4*>(dst + x * kRowBytes + ((ch ^ x) << 4)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        *reinterpret_cast<uint4*>(dst + (x + 8) * kRowBytes + ((ch ^ x) << 4)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    } else {
                        *reinterpret_cast<uint4*>(dst + x * kRowBytes + ((ch ^ (x & 7)) << 4)) = v.w;
                    }
                }
                __syncthreads();
            }
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int n = 0; n < NT; ++n) o[t][n][0] = o[t][n][1] = o[t][n][2] = o[t][n][3] = 0.f;
        }
        cp_async_wait<STAGES - 2>();
        __syncwarp();
        if (!L.done) request(stage == 0 ? STAGES - 1 : stage - 1);
        cp_async_commit();

        const uint32_t key0 = C.t * kTile + warp * 16;
        if (key0 < C.hi && key0 + 16 > C.lo) {
            const uint32_t ks0 = pipe + stage * (2 * kSlice), vs0 = ks0 + kSlice;
            float sc[MT][2][4] = {};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint32_t kb[4];
                const uint32_t r = ((lane >> 4) << 3) + (lane & 7), c = 2 * ks + ((lane >> 3) & 1);
                ldmatrix_x4(kb, ks0 + r * kRowBytes + ((c ^ (r & 7)) << 4));
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    if constexpr (MT == 1) {
                        mma<P>(sc[0][0], qf[ks], kb[0], kb[1]);
                        mma<P>(sc[0][1], qf[ks], kb[2], kb[3]);
                    } else {
                        uint32_t qa[4];
                        const uint32_t x = lane & 15, ch = 2 * ks + (lane >> 4);
                        ldmatrix_x4(qa, smem_u32(qs) + (t * 16 + x) * kRowBytes + ((ch ^ (x & 7)) << 4));
                        mma<P>(sc[t][0], qa, kb[0], kb[1]);
                        mma<P>(sc[t][1], qa, kb[2], kb[3]);
                    }
                }
            }
            uint32_t pa[MT][4];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                // w[j][n][e]: row g + 8 j of product t, key 8 n + 2 tq + e of the slice
                float w[J][2][2];
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if constexpr (SPLIT) {
                            w[0][n][e] = (sc[t][n][e] + sc[t][n][e + 2]) * p.scale_log2;
                        } else {
                            w[0][n][e] = sc[t][n][e] * p.scale_log2;
                            w[J - 1][n][e] = sc[t][n][e + 2] * p.scale_log2;
                        }
                    }
                bool grows = false;
                float top[J];
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const int32_t low = p.window != 0 ? at[t][j] - static_cast<int32_t>(min(p.window, 0x7fffffffu)) : -1;
                    const int32_t up = min(at[t][j], static_cast<int32_t>(C.hi) - 1);  // (a row's position may lie behind the last key)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int32_t key = static_cast<int32_t>(key0 + 8 * n + 2 * tq + e);
                            if (key > up || key <= low) w[j][n][e] = -INFINITY;
                        }
                    top[j] = fmaxf(fmaxf(w[j][0][0], w[j][0][1]), fmaxf(w[j][1][0], w[j][1][1]));
                    top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 1));
                    top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 2));
                    grows = grows || top[j] > m[t][j] + kRescaleStep || (m[t][j] == -INFINITY && top[j] != -INFINITY);
                }
                if (__any_sync(0xffffffffu, grows)) {
                    float f[2];
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        const float to = fmaxf(m[t][j], top[j]);
                        f[j] = m[t][j] == -INFINITY ? 0.f : fast_exp2(m[t][j] - to);
                        m[t][j] = to;
                        l[t][j] *= f[j];
                    }
                    if constexpr (SPLIT) f[1] = f[0];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        o[t][n][0] *= f[0];
                        o[t][n][1] *= f[0];
                        o[t][n][2] *= f[1];
                        o[t][n][3] *= f[1];
                    }
                }
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    // (f32 rows: lifted behind the exponential, whose argument would cost the largest weights three of their bits)
                    const float base = m[t][j] == -INFINITY ? 0.f : SPLIT ? m[t][j] : m[t][j] - kLift<P>;
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            w[j][n][e] = SPLIT ? fast_exp2(w[j][n][e] - base) * (1.f / kUnlift<P>) : fast_exp2(w[j][n][e] - base);
                            l[t][j] += w[j][n][e];
                        }
                }
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    if constexpr (SPLIT) {
                        __half h0, l0, h1, l1;
                        split_half(w[0][n][0], h0, l0);
                        split_half(w[0][n][1], h1, l1);
                        pa[t][2 * n] = pack_half2(h0, h1);
                        pa[t][2 * n + 1] = pack_half2(l0, l1);
                    } else {
                        pa[t][2 * n] = pack2(P(), w[0][n][0], w[0][n][1]);
                        pa[t][2 * n + 1] = pack2(P(), w[J - 1][n][0], w[J - 1][n][1]);
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
                uint32_t vb[4];
                const uint32_t r = lane & 15, c = n + (lane >> 4);
                ldmatrix_x4_trans(vb, vs0 + r * kRowBytes + ((c ^ (r & 7)) << 4));
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    if constexpr (SPLIT) {
                        // The tensor core cuts its sums short of a rounding, which adds up over a long cache (2e-6 of the
                        // norm at 32768 keys): a slice's products start at zero and are added here.
                        float a0[4] = {}, a1[4] = {};
                        mma<P>(a0, pa[t], vb[0], vb[1]);
                        mma<P>(a1, pa[t], vb[2], vb[3]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            o[t][n][e] += a0[e];
                            o[t][n + 1][e] += a1[e];
                        }
                    } else {
                        mma<P>(o[t][n], pa[t], vb[0], vb[1]);
                        mma<P>(o[t][n + 1], pa[t], vb[2], vb[3]);
                    }
                }
            }
        }

        if (C.t + 1 == C.t_end) {
            // ---- the run's part of the cell is complete: join the warps ----------------------------------------------
            const bool whole = C.tile0 == 0 && C.next - C.pos >= C.T;  // no other CTA has a part of the cell
            const uint64_t cell0 = C.pos - C.tile0;
            const uint32_t first = whole ? cta : static_cast<uint32_t>(cell0 / per);
            const uint32_t last = whole ? cta : static_cast<uint32_t>((cell0 + C.T - 1) / per);
            const uint32_t part = C.tile0 == 0 ? 2 * cta + 1 : 2 * cta;
            const uint32_t cols = head_dim / 4;
            auto write = [&](uint32_t pair, uint32_t c4, float4 v, float top, float sum) {
                const uint32_t abs_pair = C.b * PB + pair;
                const uint32_t row = abs_pair / group, head = C.kvh * group + abs_pair % group;
                const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
                T* dst = static_cast<T*>(p.out) + static_cast<uint64_t>(C.row0 + row) * p.out_row + head * head_dim + 4 * c4;
                const float x[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
                if constexpr (SPLIT) {
                    *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
                } else {
                    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(P(), x[0], x[1]), pack2(P(), x[2], x[3]));
                }
                if (c4 == 0 && p.lse)
                    p.lse[static_cast<uint64_t>(C.row0 + row) * p.q_heads + head] =
                        sum > 0.f || sum != sum ? (top + log2f(sum * kUnlift<P>)) * 0.69314718055994530942f : -INFINITY;
            };
            const uint32_t pairs = min(C.rows * group - C.b * PB, PB);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                // The stage just used (of every warp) holds the warp's output rows, PT x D floats; columns are twisted by
                // the row so that the eight rows a warp writes at a time spread over the banks.
                __syncwarp();
                float* const ex = reinterpret_cast<float*>(smem + warp * (STAGES * 2 * kSlice) + stage * (2 * kSlice));
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    l[t][j] += __shfl_xor_sync(0xffffffffu, l[t][j], 1);
                    l[t][j] += __shfl_xor_sync(0xffffffffu, l[t][j], 2);
                    if (tq == 0) {
                        wm[warp * 16 + g + 8 * j] = m[t][j];
                        wl[warp * 16 + g + 8 * j] = l[t][j];
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float2 x = make_float2(o[t][n][2 * j], o[t][n][2 * j + 1]);
                        if constexpr (SPLIT) x = make_float2(o[t][n][0] + o[t][n][2], o[t][n][1] + o[t][n][3]);
                        *reinterpret_cast<float2*>(ex + (g + 8 * j) * D + ((8 * n + 2 * tq) ^ (8 * (g & 7)))) = x;
                    }
                }
                __syncthreads();
                const uint32_t here = pairs > t * PT ? min(pairs - t * PT, PT) : 0u;
                for (uint32_t i = tid; i < here * cols; i += kThreads) {
                    const uint32_t x = i / cols, c4 = i % cols, pair = t * PT + x;
                    float top = wm[x];
#pragma unroll
                    for (int w = 1; w < kWarps; ++w) top = fmaxf(top, wm[w * 16 + x]);
                    float sum = 0.f;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) {
                        const float f = wm[w * 16 + x] == -INFINITY ? 0.f : fast_exp2(wm[w * 16 + x] - top);
                        sum += f * wl[w * 16 + x];
                        const float4 y = *reinterpret_cast<const float4*>(
                            reinterpret_cast<const float*>(smem + w * (STAGES * 2 * kSlice) + stage * (2 * kSlice)) + x * D +
                            ((4 * c4) ^ (8 * (x & 7))));
                        v.x += f * y.x;
                        v.y += f * y.y;
                        v.z += f * y.z;
                        v.w += f * y.w;
                    }
                    if (whole) {
                        write(pair, c4, v, top, sum);
                    } else {
                        reinterpret_cast<float4*>(p.part_o + (static_cast<size_t>(part) * kStreamRows + pair) * D)[c4] = v;
                        if (c4 == 0) reinterpret_cast<float2*>(p.part_ml)[part * kStreamRows + pair] = make_float2(top, sum);
                    }
                }
                __syncthreads();  // the stage may be filled again, and every store of the part is done
            }
            if (!whole) {
                if (tid == 0) {
                    const uint32_t ticket = take_ticket(p.tickets + first);
                    *s_flag = ticket == last - first ? 1u : 0u;
                    if (ticket == last - first) p.tickets[first] = 0u;  // as the next launch wants it
                }
                __syncthreads();
                if (*s_flag != 0u) {
                    // The parts lie in slots 2 first + 1 (where the cell begins), 2 (first + 1), 2 (first + 2), ...  A thread
                    // asks for B of them at a time: their latency is what a join costs (16 took longer again, in code to fetch).
                    auto join = [&](auto batch) {
                        constexpr int B = decltype(batch)::value;
                        for (uint32_t i = tid; i < pairs * cols; i += kThreads) {
                            const uint32_t pair = i / cols, c4 = i % cols;
                            float top = -INFINITY, sum = 0.f;
                            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                            for (uint32_t c0 = first; c0 <= last; c0 += B) {
                                float2 ml[B];
                                float4 x[B];
#pragma unroll
                                for (int u = 0; u < B; ++u) {
                                    const uint32_t c = min(c0 + u, last), slot = c == first ? 2 * c + 1 : 2 * c;
                                    ml[u] = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + slot * kStreamRows + pair);
                                    x[u] = __ldcg(reinterpret_cast<const float4*>(p.part_o + (static_cast<size_t>(slot) * kStreamRows + pair) * D) + c4);
                                }
                                float to = top;
#pragma unroll
                                for (int u = 0; u < B; ++u) to = fmaxf(to, ml[u].x);
                                const float f0 = top == -INFINITY ? 0.f : fast_exp2(top - to);
                                sum *= f0;
                                v.x *= f0, v.y *= f0, v.z *= f0, v.w *= f0;
                                top = to;
#pragma unroll
                                for (int u = 0; u < B; ++u) {
                                    const float f = c0 + u <= last && ml[u].x != -INFINITY ? fast_exp2(ml[u].x - top) : 0.f;
                                    sum += f * ml[u].y;
                                    v.x += f * x[u].x, v.y += f * x[u].y, v.z += f * x[u].z, v.w += f * x[u].w;
                                }
                            }
                            write(pair, c4, v, top, sum);
                        }
                    };
                    if (last - first < 2)
                        join(std::integral_constant<int, 2>());
                    else
                        join(std::integral_constant<int, 8>());
                    __syncthreads();  // before s_flag is written again
                }
            }
        }
        step(C);
        stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
}

template <typename T, int D, int STAGES, int MT>
cudaError_t launch_as(const AttnParams& p, uint32_t sms, cudaStream_t s) {
    auto kernel = paged_stream_kernel<T, D, STAGES, MT>;
    static OncePerDevice prepared;
    if (!prepared.done(p.device)) {
        const cudaError_t e = handled(
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem_bytes<D, STAGES>(MT, kMaxSeqs))));
        if (e != cudaSuccess) return e;
        prepared.mark(p.device);
    }
    return launch_dependent(kernel, stream_ctas(sms, p.pool.head_dim), kThreads, smem_bytes<D, STAGES>(MT, p.batch.n_seqs), s, p);
}
template <typename T>
cudaError_t launch_width(const AttnParams& p, bool wide, uint32_t sms, cudaStream_t s) {
    if (p.pool.head_dim <= 64) return wide ? launch_as<T, 64, 4, 2>(p, sms, s) : launch_as<T, 64, 4, 1>(p, sms, s);
    if (p.pool.head_dim <= 128) return wide ? launch_as<T, 128, 3, 2>(p, sms, s) : launch_as<T, 128, 3, 1>(p, sms, s);
    return launch_as<T, 256, 3, 1>(p, sms, s);  // (twice the outputs would not fit the registers)
}

}  // namespace

uint32_t stream_pairs(int32_t row_dtype) { return row_dtype == ITK_ROW_F32 ? RowTraits<float>::kPairs : RowTraits<__half>::kPairs; }

cudaError_t launch_stream(const AttnParams& p, int32_t row_dtype, bool wide, uint32_t sms, cudaStream_t s) {
    if (row_dtype == ITK_ROW_F32) return launch_width<float>(p, wide, sms, s);
    if (row_dtype == ITK_ROW_F16) return launch_width<__half>(p, wide, sms, s);
    return launch_width<__nv_bfloat16>(p, wide, sms, s);
}

}  // namespace paged
}  // namespace itk
