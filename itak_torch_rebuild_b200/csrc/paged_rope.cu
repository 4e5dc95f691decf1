// The rotation of head rows by a frequency table, alone (forward or gradient) and on the way into the pages of a cache.
//
// Pair (a, b) of channels at position p:  a' = m (a cos t - b sin t),  b' = m (a sin t + b cos t),  t = p * inv_freq[i].
// The angle is formed in f64 (at position 131072 an f32 angle is off by 2^-8) in half turns, reduced to [-1, 1] exactly,
// and only then goes to f32 and sincospif: 1e-7 absolute.  The gradient of the map is the rotation by -t.
//
// Bound: HBM for prompts - every element is read and written once - and the latency of a dependent chain (starts, length,
// page number, data) for a decode step.  One CTA owns one token (a row with all its heads), so that its angles are taken
// once, by as many threads as there are pairs, and shared through shared memory by every head; the first heads' data is
// requested before the angles are known.
//
// Measured (share of the copy rate): 8192 x 64 head rows of 128 bf16 channels 47 us (0.88), f32 82 us (1.0); 6 ragged sequences
// of 611-2048 new tokens, 64 / 8 heads, Q, K and V 57-58 us (0.88); a decode step of 16 sequences 3.5 us.
#include <math.h>

#include "paged.cuh"

namespace itk {
namespace paged {
namespace {

constexpr int kThreads = 128;  // (8192 rows x 64 heads of 128 bf16 channels: 46.5 us, with 256 threads 51.5)
constexpr int kAhead = 2;  // heads of a thread requested before the angles are there

struct RopeLaunch {
    const void* x;
    void* out;
    const uint32_t* positions;
    const double* inv_freq;
    uint64_t x_row, x_head, o_row, o_head;
    uint32_t heads, head_dim, half, pairing, items;  // items: units of work of one head (see `Item`)
    float magnitude, sign;
};

// cos and sin of pair i at position `pos`, times the magnitude.
__device__ __forceinline__ float2 turn_of(double pos, double inv_freq, float magnitude, float sign) {
    const double half_turns = pos * (inv_freq * 0.31830988618379067154);
    const float r = static_cast<float>(half_turns - 2.0 * rint(0.5 * half_turns));
    float s, c;
    sincospif(r, &s, &c);
    return make_float2(c * magnitude, s * (magnitude * sign));
}

// The unit of work `item` of a head row, eight channels wide:
//   adjacent pairs   item = channels [8 item, 8 item + 8): four pairs, those from `half` on copied
//   half split       item < half / 8: channels c = 8 item.. and their partners c + half..; later items copy the
//                    channels behind the rotated part.  Wants half and head_dim to be multiples of 8.
// `Wide` holds what one item reads.
template <typename T>
struct Wide {
    Vec8<T> a, b;
};
__device__ __forceinline__ uint32_t first_channel(uint32_t item, uint32_t half, uint32_t pairing) {
    return pairing != 0 && item >= half / 8 ? 8 * item + half : 8 * item;
}
template <typename T>
__device__ __forceinline__ void wide_load(Wide<T>& w, const T* row, uint32_t item, uint32_t half, uint32_t pairing) {
    const uint32_t c = first_channel(item, half, pairing);
    w.a.load(row + c);
    if (pairing != 0 && item < half / 8) w.b.load(row + c + half);
}
template <typename T, typename O>
__device__ __forceinline__ void copy8(const Vec8<T>& v, O* dst) {
    if constexpr (sizeof(T) == sizeof(O)) {
        v.store(dst);  // the same type: its bits
    } else {
        float f[8];
        v.get(f);
        Vec8<O> o;
        o.set(f);
        o.store(dst);
    }
}
template <typename T, typename O>
__device__ __forceinline__ void wide_turn(const Wide<T>& w, O* row, uint32_t item, uint32_t half, uint32_t pairing,
                                          const float2* cs) {
    const uint32_t c = first_channel(item, half, pairing);
    if (pairing == 0) {
        if (4 * item >= half) return copy8(w.a, row + c);
        float f[8];
        w.a.get(f);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t i = 4 * item + j;
            if (i < half) {
                const float2 t = cs[i];
                const float a = f[2 * j], b = f[2 * j + 1];
                f[2 * j] = a * t.x - b * t.y;
                f[2 * j + 1] = a * t.y + b * t.x;
            }
        }
        Vec8<O> o;
        o.set(f);
        o.store(row + c);
        return;
    }
    if (item >= half / 8) return copy8(w.a, row + c);
    float f[8], g[8];
    w.a.get(f);
    w.b.get(g);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float2 t = cs[c + j];
        const float a = f[j], b = g[j];
        f[j] = a * t.x - b * t.y;
        g[j] = a * t.y + b * t.x;
    }
    Vec8<O> o;
    o.set(f);
    o.store(row + c);
    o.set(g);
    o.store(row + c + half);
}
// How a kernel goes through a head row: kWide as above; kWhole for half-split pairs whose halves are not multiples of eight
// channels - a warp takes whole rows (as many as its lanes cover, eight channels a lane) by way of shared memory, where
// partners lie at any distance (8192 x 64 rows of 62 rotated channels: 178 us pair by pair); kNarrow, one pair or one copied channel at
// a time, for rows that 16-byte words cannot address.
enum Mode { kWide, kWhole, kNarrow };
constexpr int kWarps = kThreads / 32;

// Lanes of kWhole read eight elements apart: one place more for every eight spreads them over the banks.
__device__ __forceinline__ uint32_t skew(uint32_t i) { return i + i / 8; }
constexpr uint32_t kSkewedDim = kMaxHeadDim + kMaxHeadDim / 8;

// Lane `item` of a row's head_dim / 8; `row` holds the head row in f32.  The whole warp calls it, `active` lanes work.
template <typename T, typename O>
__device__ __forceinline__ void whole_turn(const T* src, O* dst, bool active, uint32_t item, uint32_t half, const float2* cs, float* row) {
    Vec8<T> v = {};
    float f[8];
    if (active) {
        v.load(src + 8 * item);
        v.get(f);
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) row[skew(8 * item) + j] = f[j];
    }
    __syncwarp();
    if (active) {
        if (8 * item >= 2 * half) {
            copy8(v, dst + 8 * item);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
                const uint32_t c = 8 * item + j;
                const bool first = c < half;
                if (c < 2 * half) {
                    const float2 t = cs[skew(first ? c : c - half)];
                    const float other = row[skew(first ? c + half : c - half)];
                    f[j] = f[j] * t.x + (first ? -other : other) * t.y;
                }
            }
            Vec8<O> o;
            o.set(f);
            o.store(dst + 8 * item);
        }
    }
    __syncwarp();
}

template <typename T, typename O>
__device__ __forceinline__ void narrow_turn(const T* src, O* dst, uint32_t item, uint32_t half, uint32_t pairing,
                                            const float2* cs) {
    if (item < half) {
        const uint32_t a = pairing == 0 ? 2 * item : item, b = pairing == 0 ? 2 * item + 1 : item + half;
        const float2 t = cs[item];
        const float u = to_f32(src[a]), v = to_f32(src[b]);
        dst[a] = from_f32<O>(u * t.x - v * t.y);
        dst[b] = from_f32<O>(u * t.y + v * t.x);
    } else {
        if constexpr (sizeof(T) == sizeof(O))
            dst[item + half] = src[item + half];
        else
            dst[item + half] = from_f32<O>(to_f32(src[item + half]));
    }
}

template <typename T, Mode M>
__global__ void __launch_bounds__(kThreads) rope_apply_kernel(const __grid_constant__ RopeLaunch p) {
    __shared__ float2 cs[kSkewedDim / 2];
    __shared__ float whole[M == kWhole ? kWarps : 1][M == kWhole ? kSkewedDim : 1];
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const uint32_t step = max(kThreads / p.items, 1u);  // heads the CTA works on at a time (one, when it has more items than threads)
    const uint32_t item = tid % p.items, h0 = tid / p.items;
    const T* src = static_cast<const T*>(p.x) + row * p.x_row;
    T* dst = static_cast<T*>(p.out) + row * p.o_row;
    Wide<T> ahead[kAhead];
    after_predecessor();
    if constexpr (M == kWide) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (h0 < step && h0 + j * step < p.heads) wide_load(ahead[j], src + (h0 + j * step) * p.x_head, item, p.half, p.pairing);
    }
    const double pos = static_cast<double>(p.positions[row]);
    for (uint32_t i = tid; i < p.half; i += kThreads) cs[M == kWhole ? skew(i) : i] = turn_of(pos, p.inv_freq[i], p.magnitude, p.sign);
    __syncthreads();
    if constexpr (M == kWhole) {
        const uint32_t lane = tid & 31, at_once = 32 / p.items, sub = lane / p.items, u = lane % p.items;
        for (uint32_t first = (tid >> 5) * at_once; first < p.heads; first += kWarps * at_once) {
            const uint32_t h = first + sub;
            whole_turn(src + h * p.x_head, dst + h * p.o_head, sub < at_once && h < p.heads, u, p.half, cs, whole[tid >> 5] + (sub < at_once ? sub : 0u) * skew(p.head_dim));
        }
        return;
    }
    if (h0 >= step) return;
    if constexpr (M == kWide) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (h0 + j * step < p.heads) wide_turn(ahead[j], dst + (h0 + j * step) * p.o_head, item, p.half, p.pairing, cs);
        for (uint32_t h = h0 + kAhead * step; h < p.heads; h += step) {
            Wide<T> w;
            wide_load(w, src + h * p.x_head, item, p.half, p.pairing);
            wide_turn(w, dst + h * p.o_head, item, p.half, p.pairing, cs);
        }
    } else {
        for (uint32_t h = h0; h < p.heads; h += step)
            for (uint32_t u = item; u < p.items; u += kThreads) narrow_turn(src + h * p.x_head, dst + h * p.o_head, u, p.half, p.pairing, cs);
    }
}

struct AppendRows {
    Pool pool;
    Batch batch;
    const void* q;
    void* q_out;
    const void* k;
    const void* v;
    const double* inv_freq;
    uint64_t q_row, q_out_row, k_row, v_row;
    uint32_t q_heads, half, pairing, items;
    float magnitude;
};

// T: rows, P: pages.  Heads are counted through: the q_heads of q first (none without q), then K's, then V's.
template <typename T, typename P, Mode M>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const __grid_constant__ AppendRows p) {
    __shared__ float2 cs[kSkewedDim / 2];
    __shared__ float whole[M == kWhole ? kWarps : 1][M == kWhole ? kSkewedDim : 1];
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const uint32_t D = p.pool.head_dim, hq = p.q_heads, hkv = p.pool.kv_heads;
    const uint32_t heads = hq + 2 * hkv;
    const uint32_t step = max(kThreads / p.items, 1u);
    const uint32_t item = tid % p.items, h0 = tid / p.items;
    const T* q = static_cast<const T*>(p.q) + row * p.q_row;
    const T* k = static_cast<const T*>(p.k) + row * p.k_row;
    const T* v = static_cast<const T*>(p.v) + row * p.v_row;
    auto source = [&](uint32_t h) { return h < hq ? q + h * D : h < hq + hkv ? k + (h - hq) * D : v + (h - hq - hkv) * D; };
    Wide<T> ahead[kAhead];
    after_predecessor();
    if constexpr (M == kWide) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (h0 < step && h0 + j * step < heads) wide_load(ahead[j], source(h0 + j * step), item, p.half, p.pairing);
    }
    // The row's sequence: as many starts s + 1 as lie at or before the row.
    uint32_t seq = 0;
    for (uint32_t s0 = 0; s0 < p.batch.n_seqs; s0 += kThreads) {
        const uint32_t s = s0 + tid;
        const bool before = s < p.batch.n_seqs && p.batch.row_start[s + 1] <= row;
        seq += __syncthreads_count(before);
    }
    if (row == 0 && p.batch.status != nullptr)  // one CTA looks the batch over
        for (uint32_t s = tid; s < p.batch.n_seqs; s += kThreads) seq_of(p.batch, s, p.pool.page_shift);
    if (seq >= p.batch.n_seqs) return;  // behind the last sequence
    const Seq sq = seq_of(Batch{p.batch.table, p.batch.row_start, p.batch.kv_len, nullptr, p.batch.n_seqs, p.batch.table_width,
                                p.batch.table_stride, p.batch.total_rows}, seq, p.pool.page_shift);
    if (row < sq.row0 || row - sq.row0 >= sq.rows) return;
    const int32_t pos = sq.pos0 + static_cast<int32_t>(row - sq.row0);
    if (pos < 0) return;
    // A row behind the table's last column has no place (reported with its sequence); its query is turned all the same.
    const bool placed = static_cast<uint32_t>(pos) < room_of(p.batch, p.pool.page_shift);
    const uint32_t page = placed ? p.batch.table[static_cast<size_t>(seq) * p.batch.table_stride + (static_cast<uint32_t>(pos) >> p.pool.page_shift)] : 0u;
    const bool stored = placed && page < p.pool.n_pages;
    if (placed && !stored && tid == 0) raise(p.batch, kBadPage);
    const uint64_t at = page * p.pool.page_stride + (static_cast<uint32_t>(pos) & ((1u << p.pool.page_shift) - 1u)) * p.pool.row_stride;
    P* const kp = static_cast<P*>(p.pool.k) + at;
    P* const vp = static_cast<P*>(p.pool.v) + at;
    T* const qo = static_cast<T*>(p.q_out) + row * p.q_out_row;
    for (uint32_t i = tid; i < p.half; i += kThreads) cs[M == kWhole ? skew(i) : i] = turn_of(static_cast<double>(pos), p.inv_freq[i], p.magnitude, 1.f);
    __syncthreads();
    if constexpr (M == kWhole) {
        const uint32_t lane = tid & 31, at_once = 32 / p.items, sub = lane / p.items, u = lane % p.items;
        float* const mine = whole[tid >> 5] + (sub < at_once ? sub : 0u) * skew(D);
        const uint32_t turned = hq + hkv;
        for (uint32_t first = (tid >> 5) * at_once; first < turned; first += kWarps * at_once) {  // (Q and K rows in one go: a
            const uint32_t h = first + sub;                                                      // warp's rows may be of both)
            const bool active = sub < at_once && h < turned && (h < hq || stored);
            if constexpr (sizeof(T) == sizeof(P)) {
                whole_turn(source(h < turned ? h : 0u), h < hq ? reinterpret_cast<P*>(qo + h * D) : kp + (h - hq) * p.pool.head_stride, active, u, p.half, cs, mine);
            } else {
                whole_turn(source(h < turned ? h : 0u), qo + h * D, active && h < hq, u, p.half, cs, mine);
                whole_turn(source(h < turned ? h : 0u), kp + (h - hq) * p.pool.head_stride, active && h >= hq, u, p.half, cs, mine);
            }
        }
        if (stored)
            for (uint32_t i = tid; i < hkv * p.items; i += kThreads) {
                Vec8<T> x;
                x.load(v + 8 * i);  // (a token's heads are contiguous)
                copy8(x, vp + (i / p.items) * p.pool.head_stride + 8 * (i % p.items));
            }
        return;
    }
    if (h0 >= step) return;
    auto put = [&](uint32_t h, const Wide<T>& w) {
        if (h < hq) {
            wide_turn(w, qo + h * D, item, p.half, p.pairing, cs);
        } else if (stored) {
            if (h < hq + hkv) {
                wide_turn(w, kp + (h - hq) * p.pool.head_stride, item, p.half, p.pairing, cs);
            } else {
                const uint32_t c = first_channel(item, p.half, p.pairing);
                P* dst = vp + (h - hq - hkv) * p.pool.head_stride;
                copy8(w.a, dst + c);
                if (p.pairing != 0 && item < p.half / 8) copy8(w.b, dst + c + p.half);
            }
        }
    };
    if constexpr (M == kWide) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (h0 + j * step < heads) put(h0 + j * step, ahead[j]);
        for (uint32_t h = h0 + kAhead * step; h < heads; h += step) {
            Wide<T> w;
            wide_load(w, source(h), item, p.half, p.pairing);
            put(h, w);
        }
    } else {
        for (uint32_t h = h0; h < heads; h += step) {
            const T* src = source(h);
            if (h < hq + hkv) {
                if (h >= hq && !stored) continue;
                for (uint32_t u = item; u < p.items; u += kThreads) {
                    if (h < hq)
                        narrow_turn(src, qo + h * D, u, p.half, p.pairing, cs);
                    else
                        narrow_turn(src, kp + (h - hq) * p.pool.head_stride, u, p.half, p.pairing, cs);
                }
            } else if (stored) {
                P* dst = vp + (h - hq - hkv) * p.pool.head_stride;
                const uint32_t across = min(p.items, static_cast<uint32_t>(kThreads));
                for (uint32_t c = item; c < D; c += across) {
                    if constexpr (sizeof(T) == sizeof(P))
                        dst[c] = src[c];
                    else
                        dst[c] = from_f32<P>(to_f32(src[c]));
                }
            }
        }
    }
}

// The way through rows that sixteen-byte words can address or not, and its items per head row.
Mode mode_of(bool words, uint32_t head_dim, uint32_t half, uint32_t pairing) {
    if (!words || head_dim % 8 != 0) return kNarrow;
    return pairing == 0 || half % 8 == 0 ? kWide : kWhole;
}
uint32_t items_of(Mode m, uint32_t head_dim, uint32_t half, uint32_t pairing) {
    if (m == kNarrow) return half + (head_dim - 2 * half);
    return m == kWide && pairing != 0 ? half / 8 + (head_dim - 2 * half) / 8 : head_dim / 8;
}

}  // namespace

int check_pool(const itk_paged_kv* kv, const ErrorText& e, Pool* out) {
    if (!kv) return e.invalid("null pointer argument");
    if (kv->kv_heads == 0) return e.refuse(ITK_ERR_ZERO_DIMENSION, "num_kv_heads must be positive, got 0");
    if (kv->head_dim == 0) return e.refuse(ITK_ERR_ZERO_DIMENSION, "head_dim must be positive, got 0");
    if (kv->n_pages == 0) return e.refuse(ITK_ERR_ZERO_DIMENSION, "n_pages must be positive, got 0");
    if (kv->head_dim % 8 != 0 || kv->head_dim > kMaxHeadDim)
        return e.invalid("head_dim %llu must be a multiple of 8 up to %llu", kv->head_dim, kMaxHeadDim);
    if (kv->page_size == 0 || kv->page_size > 65536 || (kv->page_size & (kv->page_size - 1)) != 0)
        return e.invalid("page_size %llu must be a power of two up to 65536", kv->page_size);
    if (kv->dtype != ITK_ROW_F16 && kv->dtype != ITK_ROW_BF16) return e.invalid("pages hold ITK_ROW_F16 or ITK_ROW_BF16");
    if (kv->kv_heads > 65535) return e.invalid("kv_heads %llu is too large", kv->kv_heads);
    if (kv->n_pages > 0x7fffffffu) return e.invalid("n_pages %llu is too large", kv->n_pages);
    if (!kv->k || !kv->v) return e.invalid("null pointer argument");
    if (!aligned16(kv->k) || !aligned16(kv->v)) return e.invalid("the pools must start on a 16-byte boundary");
    const uint64_t st[3] = {kv->page_stride, kv->head_stride, kv->row_stride};
    for (uint64_t s : st)
        if (s % 8 != 0 || s >= kMaxStride) return e.invalid("page strides must be multiples of 8 elements, got %llu", s);
    // rows and heads must not share elements: whichever of the two is the outer one steps over all of the inner one
    const uint64_t D = kv->head_dim, row_span = (kv->page_size - 1ull) * kv->row_stride + D, head_span = (kv->kv_heads - 1ull) * kv->head_stride + D;
    const bool rows_inside = (kv->page_size == 1 || kv->row_stride >= D) && (kv->kv_heads == 1 || kv->head_stride >= row_span);
    const bool heads_inside = (kv->kv_heads == 1 || kv->head_stride >= D) && (kv->page_size == 1 || kv->row_stride >= head_span);
    if (!rows_inside && !heads_inside) return e.invalid("rows and heads of a page overlap (head stride %llu, row stride %llu)", kv->head_stride, kv->row_stride);
    if (kv->n_pages > 1 && kv->page_stride < (kv->page_size - 1ull) * kv->row_stride + (kv->kv_heads - 1ull) * kv->head_stride + D)
        return e.invalid("pages overlap (page stride %llu)", kv->page_stride);
    out->k = kv->k;
    out->v = kv->v;
    out->page_stride = kv->page_stride;
    out->head_stride = kv->head_stride;
    out->row_stride = kv->row_stride;
    out->n_pages = kv->n_pages;
    out->page_shift = static_cast<uint32_t>(__builtin_ctz(kv->page_size));
    out->kv_heads = kv->kv_heads;
    out->head_dim = kv->head_dim;
    return 0;
}

int check_batch(const itk_paged_batch* b, const ErrorText& e, Batch* out) {
    if (!b || !b->table || !b->row_start || !b->kv_len) return e.invalid("null pointer argument");
    if (b->n_seqs == 0) return e.refuse(ITK_ERR_ZERO_DIMENSION, "n_seqs must be positive, got 0");
    if (b->n_seqs > kMaxSeqs) return e.refuse(ITK_ERR_CAPACITY, "%llu sequences in one batch, at most %llu", b->n_seqs, kMaxSeqs);
    if (b->table_width == 0) return e.refuse(ITK_ERR_ZERO_DIMENSION, "table_width must be positive, got 0");
    if (b->table_stride < b->table_width && b->n_seqs > 1)
        return e.invalid("table_stride %llu is shorter than table_width %llu", b->table_stride, b->table_width);
    if (!aligned_to(b->table, 4) || !aligned_to(b->row_start, 4) || !aligned_to(b->kv_len, 4) || !aligned_to(b->status, 4))
        return e.invalid("table, row_start, kv_len and status must be aligned to 4 bytes");
    if (b->total_rows > 0x7fffffffu) return e.invalid("total_rows %llu is too large", b->total_rows);
    out->table = b->table;
    out->row_start = b->row_start;
    out->kv_len = b->kv_len;
    out->status = b->status;
    out->n_seqs = b->n_seqs;
    out->table_width = b->table_width;
    out->table_stride = b->table_stride;
    out->total_rows = b->total_rows;
    return 0;
}

int check_row_dtype(int32_t rows, int32_t pages, const ErrorText& e) {
    if (rows != ITK_ROW_F32 && rows != ITK_ROW_F16 && rows != ITK_ROW_BF16) return e.invalid("unknown element type %llu of the rows", static_cast<unsigned long long>(rows));
    if ((rows == ITK_ROW_BF16) != (pages == ITK_ROW_BF16))
        return e.invalid("f32 and f16 rows go with f16 pages, bf16 rows with bf16 pages");
    return 0;
}

}  // namespace paged
}  // namespace itk

extern "C" int itk_rope_table(const itk_rope_config* c, double* inv_freq, float* magnitude, char* error_text, size_t error_text_len) {
    using namespace itk::paged;
    const ErrorText e(error_text, error_text_len);
    if (!c || !inv_freq || !magnitude) return e.invalid("null pointer argument");
    if (c->rotary_dim < 2 || c->rotary_dim % 2 != 0 || c->rotary_dim > kMaxHeadDim)
        return e.invalid("rope: rotary_dim %llu must be even and in 2..%llu", c->rotary_dim, kMaxHeadDim);
    if (!(c->base > 1.0f) || !isfinite(c->base)) return e.invalid("rope: base must be finite and > 1");
    if (c->scaling < ITK_ROPE_PLAIN || c->scaling > ITK_ROPE_PAIRS) return e.invalid("rope: unknown scaling %llu", static_cast<unsigned long long>(c->scaling));
    if (!(c->magnitude >= 0.0f) || !isfinite(c->magnitude)) return e.invalid("rope: magnitude must be finite and not negative");
    const bool by_factor = c->scaling != ITK_ROPE_PLAIN && c->scaling != ITK_ROPE_PAIRS;
    const bool banded = c->scaling == ITK_ROPE_BANDS || c->scaling == ITK_ROPE_RAMP;
    if (by_factor && (!(c->factor >= 1.0f) || !isfinite(c->factor))) return e.invalid("rope: factor must be finite and at least 1");
    if (c->scaling == ITK_ROPE_BASE && c->rotary_dim == 2) return e.invalid("rope: a scaled base needs at least two pairs");
    if (banded && (!(c->original_context > 0.0f) || !isfinite(c->original_context)))
        return e.invalid("rope: original_context must be finite and positive");
    if (banded && (!(c->low > 0.0f) || !(c->high > c->low) || !isfinite(c->high))) return e.invalid("rope: turns must satisfy 0 < low < high");
    const uint32_t half = c->rotary_dim / 2;
    if (c->scaling == ITK_ROPE_PAIRS) {
        if (!c->pair_factors) return e.invalid("null pointer argument");
        for (uint32_t i = 0; i < half; ++i)
            if (!(c->pair_factors[i] > 0.0f) || !isfinite(c->pair_factors[i])) return e.invalid("rope: the factor of pair %llu must be finite and positive", i);
    }
    const double rot = c->rotary_dim, factor = c->factor, two_pi = 6.283185307179586476925;
    double base = c->base;
    if (c->scaling == ITK_ROPE_BASE) base *= pow(factor, rot / (rot - 2.0));
    // RAMP: the pair that makes t turns over the original context, base^(-2i / rot) * original_context = 2 pi t.  The pair of
    // `low` turns may lie behind the last one (up to rot - 1): then the ramp ends before it has come down to 1 / factor.
    const double pair_span = rot / (2.0 * log(base));
    const double ramp_lo = banded ? fmax(0.0, floor(pair_span * log(c->original_context / (c->high * two_pi)))) : 0.0;
    const double ramp_hi = banded ? fmin(rot - 1.0, ceil(pair_span * log(c->original_context / (c->low * two_pi)))) : 0.0;
    for (uint32_t i = 0; i < half; ++i) {
        double f = pow(base, -2.0 * i / rot);
        double keep = 1.0;
        if (c->scaling == ITK_ROPE_LINEAR) {
            keep = 0.0;
        } else if (c->scaling == ITK_ROPE_BANDS) {
            const double turns = c->original_context * f / two_pi;
            keep = fmin(1.0, fmax(0.0, (turns - c->low) / (static_cast<double>(c->high) - c->low)));
        } else if (c->scaling == ITK_ROPE_RAMP) {
            keep = 1.0 - fmin(1.0, fmax(0.0, (i - ramp_lo) / fmax(ramp_hi - ramp_lo, 1e-3)));
        }
        if (keep < 1.0) f *= keep + (1.0 - keep) / factor;
        if (c->scaling == ITK_ROPE_PAIRS) f /= c->pair_factors[i];
        inv_freq[i] = f;
    }
    *magnitude = c->magnitude != 0.0f ? c->magnitude : c->scaling == ITK_ROPE_RAMP ? static_cast<float>(0.1 * log(factor) + 1.0) : 1.0f;
    return 0;
}

extern "C" int itk_rope_apply(const itk_rope_desc* d, void* cuda_stream, char* error_text, size_t error_text_len) {
    using namespace itk::paged;
    const ErrorText e(error_text, error_text_len);
    if (!d) return e.invalid("null pointer argument");
    if (d->rows == 0 || d->heads == 0) return e.invalid("rotate needs at least one row and head, got rows %llu, heads %llu", d->rows, d->heads);
    if (d->head_dim < 2 || d->head_dim % 2 != 0 || d->head_dim > kMaxHeadDim)
        return e.invalid("head_dim %llu must be even and in 2..%llu", d->head_dim, kMaxHeadDim);
    if (d->rotary_dim < 2 || d->rotary_dim % 2 != 0 || d->rotary_dim > d->head_dim)
        return e.invalid("rope: rotary_dim must be even, >= 2, and <= head_dim");
    if (d->pairing > 1) return e.invalid("rope: pairing is 0 (adjacent) or 1 (half split)");
    if (d->dtype != ITK_ROW_F32 && d->dtype != ITK_ROW_F16 && d->dtype != ITK_ROW_BF16) return e.invalid("unknown element type %llu of the rows", static_cast<unsigned long long>(d->dtype));
    if (!isfinite(d->magnitude)) return e.invalid("rope: magnitude must be finite");
    if (!d->x || !d->out || !d->positions || !d->inv_freq) return e.invalid("null pointer argument");
    if (!aligned_to(d->positions, 4) || !aligned_to(d->inv_freq, 8)) return e.invalid("positions must be aligned to 4 bytes and inv_freq to 8");
    if (d->rows > 0x7fffffffu) return e.invalid("rows = %llu is too large", d->rows);
    const uint64_t st[4] = {d->x_row_stride, d->x_head_stride, d->out_row_stride, d->out_head_stride};
    for (uint64_t s : st)
        if (s >= kMaxStride) return e.invalid("row stride %llu is too large", s);
    const uintptr_t size = d->dtype == ITK_ROW_F32 ? 4 : 2;
    if ((reinterpret_cast<uintptr_t>(d->x) | reinterpret_cast<uintptr_t>(d->out)) % size != 0) return e.invalid("rows must be aligned to their element type");
    const uint64_t D = d->head_dim, R = d->rows, H = d->heads;
    const bool heads_inside = (H == 1 || d->out_head_stride >= D) && (R == 1 || d->out_row_stride >= (H - 1) * d->out_head_stride + D);
    const bool rows_inside = (R == 1 || d->out_row_stride >= D) && (H == 1 || d->out_head_stride >= (R - 1) * d->out_row_stride + D);
    if (!heads_inside && !rows_inside) return e.invalid("rows of out overlap (row stride %llu, head stride %llu)", d->out_row_stride, d->out_head_stride);
    if (d->x == d->out && ((R > 1 && d->x_row_stride != d->out_row_stride) || (H > 1 && d->x_head_stride != d->out_head_stride)))
        return e.invalid("a rotation in place needs the strides of x and out to be the same");
    const uint32_t half = d->rotary_dim / 2;
    // Sixteen-byte words: every row starts on one.
    const bool words = aligned16(d->x) && aligned16(d->out) && ((R == 1 ? 0 : st[0] | st[2]) | (H == 1 ? 0 : st[1] | st[3])) % 8 == 0;
    const Mode mode = mode_of(words, d->head_dim, half, d->pairing);
    RopeLaunch p{};
    p.x = d->x;
    p.out = d->out;
    p.positions = d->positions;
    p.inv_freq = d->inv_freq;
    p.x_row = st[0];
    p.x_head = st[1];
    p.o_row = st[2];
    p.o_head = st[3];
    p.heads = d->heads;
    p.head_dim = d->head_dim;
    p.half = half;
    p.pairing = d->pairing;
    p.items = items_of(mode, d->head_dim, half, d->pairing);
    p.magnitude = d->magnitude;
    p.sign = d->inverse ? -1.f : 1.f;
    const DeviceScope scope(d->device);
    if (scope.err != cudaSuccess) return e.cuda("rotate: the device cannot be used", scope.err);
    const cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    cudaError_t err = cudaSuccess;
    auto launch = [&](auto kernel) { err = launch_dependent(kernel, d->rows, kThreads, 0, s, p); };
    auto by_mode = [&](auto row) {
        using T = decltype(row);
        mode == kWide ? launch(rope_apply_kernel<T, kWide>) : mode == kWhole ? launch(rope_apply_kernel<T, kWhole>) : launch(rope_apply_kernel<T, kNarrow>);
    };
    d->dtype == ITK_ROW_F32 ? by_mode(float()) : d->dtype == ITK_ROW_F16 ? by_mode(__half()) : by_mode(__nv_bfloat16());
    return err == cudaSuccess ? 0 : e.cuda("rotate launch failed", err);
}

extern "C" int itk_paged_append(const itk_paged_kv* kv, const itk_paged_batch* batch, const itk_paged_append_desc* d,
                                void* cuda_stream, char* error_text, size_t error_text_len) {
    using namespace itk::paged;
    const ErrorText e(error_text, error_text_len);
    AppendRows p{};
    if (int rc = check_pool(kv, e, &p.pool)) return rc;
    if (int rc = check_batch(batch, e, &p.batch)) return rc;
    if (!d) return e.invalid("null pointer argument");
    if (int rc = check_row_dtype(d->dtype, kv->dtype, e)) return rc;
    if (!d->k_new || !d->v_new) return e.invalid("null pointer argument");
    const bool with_q = d->q != nullptr;
    if (with_q != (d->q_out != nullptr) || with_q != (d->q_heads != 0)) return e.invalid("q, q_out and q_heads go together");
    if (d->q_heads > 65535) return e.invalid("q_heads %llu is too large", d->q_heads);
    const uint32_t rot = d->inv_freq ? d->rotary_dim : 0u;
    if (rot % 2 != 0 || rot > kv->head_dim) return e.invalid("rope: rotary_dim must be even and <= head_dim");
    if (d->pairing > 1) return e.invalid("rope: pairing is 0 (adjacent) or 1 (half split)");
    if (!isfinite(d->magnitude)) return e.invalid("rope: magnitude must be finite");
    if (!aligned_to(d->inv_freq, 8)) return e.invalid("inv_freq must be aligned to 8 bytes");
    const uintptr_t size = d->dtype == ITK_ROW_F32 ? 4 : 2;
    const uintptr_t starts = reinterpret_cast<uintptr_t>(d->k_new) | reinterpret_cast<uintptr_t>(d->v_new) |
                             reinterpret_cast<uintptr_t>(d->q) | reinterpret_cast<uintptr_t>(d->q_out);
    if (starts % size != 0) return e.invalid("rows must be aligned to their element type");
    const uint64_t q_width = static_cast<uint64_t>(d->q_heads) * kv->head_dim;
    const uint64_t st[4] = {d->k_row_stride, d->v_row_stride, with_q ? d->q_row_stride : 0, with_q ? d->q_out_row_stride : 0};
    for (uint64_t s : st)
        if (s >= kMaxStride) return e.invalid("row stride %llu is too large", s);
    if (batch->total_rows > 1 && with_q && d->q_out_row_stride < q_width)
        return e.invalid("rows of q_out overlap (row stride %llu, %llu elements)", d->q_out_row_stride, q_width);
    if (with_q && d->q == d->q_out && batch->total_rows > 1 && d->q_row_stride != d->q_out_row_stride)
        return e.invalid("a rotation in place needs the strides of q and q_out to be the same");
    if (batch->total_rows == 0) return 0;
    p.q = d->q;
    p.q_out = d->q_out;
    p.k = d->k_new;
    p.v = d->v_new;
    p.inv_freq = d->inv_freq;
    p.q_row = st[2];
    p.q_out_row = st[3];
    p.k_row = st[0];
    p.v_row = st[1];
    p.q_heads = d->q_heads;
    p.half = rot / 2;
    p.pairing = d->pairing;
    p.magnitude = d->magnitude;
    const bool words = starts % 16 == 0 && (batch->total_rows == 1 || (st[0] | st[1] | st[2] | st[3]) % 8 == 0);
    const Mode mode = mode_of(words, kv->head_dim, p.half, p.pairing);
    p.items = items_of(mode, kv->head_dim, p.half, p.pairing);
    const DeviceScope scope(kv->device);
    if (scope.err != cudaSuccess) return e.cuda("paged append: the device cannot be used", scope.err);
    const cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    cudaError_t err = cudaSuccess;
    auto launch = [&](auto kernel) { err = launch_dependent(kernel, batch->total_rows, kThreads, 0, s, p); };
    auto by_mode = [&](auto row, auto page) {
        using T = decltype(row);
        using P = decltype(page);
        mode == kWide ? launch(paged_append_kernel<T, P, kWide>) : mode == kWhole ? launch(paged_append_kernel<T, P, kWhole>) : launch(paged_append_kernel<T, P, kNarrow>);
    };
    d->dtype == ITK_ROW_F32 ? by_mode(float(), __half()) : d->dtype == ITK_ROW_F16 ? by_mode(__half(), __half()) : by_mode(__nv_bfloat16(), __nv_bfloat16());
    return err == cudaSuccess ? 0 : e.cuda("paged append launch failed", err);
}
