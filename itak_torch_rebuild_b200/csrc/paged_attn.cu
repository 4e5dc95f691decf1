// Host side of attention over pages: refusals, the workspace, and which kernel takes a call.
#include <math.h>

#include <atomic>

#include "paged.cuh"

namespace itk {
namespace paged {
namespace {

// Multiprocessors of a device, asked for once.
cudaError_t multiprocessors(int device, uint32_t* sms) {
    static std::atomic<uint32_t> known[64];
    if (device >= 0 && device < 64 && (*sms = known[device].load(std::memory_order_relaxed)) != 0) return cudaSuccess;
    int n = 0;
    const cudaError_t e = handled(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device));
    if (e != cudaSuccess) return e;
    *sms = static_cast<uint32_t>(n);
    if (device >= 0 && device < 64) known[device].store(*sms, std::memory_order_relaxed);
    return cudaSuccess;
}

// The bound of the tensor-memory kernel's waits: about a second unless itk_paged_attention_wait_limit says otherwise.
constexpr long long kWaitClocks = 2000000000ll;
std::atomic<uint32_t> wait_kclocks{0};

constexpr uint64_t kAlign = 256;
uint64_t round_up(uint64_t n) { return (n + kAlign - 1) / kAlign * kAlign; }

// The workspace: tickets (one per persistent CTA), then the parts' (maximum, sum) pairs, then their outputs.  A CTA
// leaves at most two parts: of the cell its run begins in and of the one it ends in.
struct Layout {
    uint64_t ml, o, bytes;
};
Layout layout_of(uint32_t sms) {
    Layout l;
    // Two parts of 256 rows for each of the tensor-memory kernel's CTAs, one per multiprocessor; the streaming kernel's
    // twice as many CTAs (above 128 channels: as many, of twice the width) have parts of 32 rows.
    const uint64_t rows = 2ull * sms * kTcRows;
    static_assert(2 * kStreamRows <= kTcRows, "the larger of the two");
    l.ml = round_up(sizeof(unsigned int) * 2ull * sms);
    l.o = l.ml + round_up(rows * 2 * sizeof(float));
    l.bytes = l.o + round_up(rows * kTcWidth * sizeof(float));
    return l;
}

}  // namespace
}  // namespace paged
}  // namespace itk

extern "C" uint64_t itk_paged_attention_workspace(int32_t device) {
    uint32_t sms = 0;
    if (itk::paged::multiprocessors(device, &sms) != cudaSuccess) return 0;
    return itk::paged::layout_of(sms).bytes;
}

extern "C" int itk_paged_attention_wait_limit(uint32_t kclocks) {
    if (kclocks > 1u << 22) return ITK_ERR_INVALID_ARGUMENT;
    itk::paged::wait_kclocks.store(kclocks, std::memory_order_relaxed);
    return 0;
}

extern "C" int itk_paged_attention(const itk_paged_kv* kv, const itk_paged_batch* batch, const itk_paged_attention_desc* d,
                                   void* cuda_stream, char* error_text, size_t error_text_len) {
    using namespace itk::paged;
    const ErrorText e(error_text, error_text_len);
    AttnParams p{};
    if (int rc = check_pool(kv, e, &p.pool)) return rc;
    if (int rc = check_batch(batch, e, &p.batch)) return rc;
    if (!d) return e.invalid("null pointer argument");
    if (int rc = check_row_dtype(d->dtype, kv->dtype, e)) return rc;
    if (d->q_heads == 0) return e.refuse(ITK_ERR_ZERO_DIMENSION, "num_q_heads must be positive, got 0");
    if (d->q_heads % kv->kv_heads != 0)
        return e.refuse(ITK_ERR_NON_DIVISIBLE_HEADS, "%llu query heads do not divide evenly across %llu KV heads", d->q_heads, kv->kv_heads);
    if (d->q_heads > 65535) return e.invalid("q_heads %llu is too large", d->q_heads);
    if (static_cast<uint64_t>(batch->total_rows) * d->q_heads > 0x7fffffffull)
        return e.invalid("total_rows x q_heads = %llu is too large", static_cast<uint64_t>(batch->total_rows) * d->q_heads);
    const float scale_log2 = static_cast<float>(static_cast<double>(d->scale) * 1.4426950408889634074);
    if (!isfinite(scale_log2)) return e.invalid("the scale must be finite, and below 2e38");
    if (!d->q || !d->out || !d->workspace) return e.invalid("null pointer argument");
    if (!aligned_to(d->lse, 4)) return e.invalid("lse must be aligned to 4 bytes");
    if (!aligned16(d->q) || !aligned16(d->out)) return e.invalid("q and out must start on a 16-byte boundary");
    const uint64_t width = static_cast<uint64_t>(d->q_heads) * kv->head_dim;
    if (d->q_row_stride % 8 != 0 || d->out_row_stride % 8 != 0 || d->q_row_stride >= kMaxStride || d->out_row_stride >= kMaxStride)
        return e.invalid("row strides must be multiples of 8 elements, got %llu and %llu", d->q_row_stride, d->out_row_stride);
    if (batch->total_rows > 1 && d->out_row_stride < width)
        return e.invalid("rows of out overlap (row stride %llu, %llu elements)", d->out_row_stride, width);
    if (reinterpret_cast<uintptr_t>(d->workspace) % kAlign != 0) return e.invalid("the workspace must start on a 256-byte boundary");
    const DeviceScope scope(kv->device);
    if (scope.err != cudaSuccess) return e.cuda("paged attention: the device cannot be used", scope.err);
    uint32_t sms = 0;
    const cudaError_t known = multiprocessors(kv->device, &sms);
    if (known != cudaSuccess) return e.cuda("paged attention: the device cannot be used", known);
    const Layout l = layout_of(sms);
    if (d->workspace_bytes < l.bytes) return e.refuse(ITK_ERR_CAPACITY, "the workspace holds %llu bytes, %llu are needed", d->workspace_bytes, l.bytes);
    if (batch->total_rows == 0) return 0;
    p.device = kv->device;
    p.q = d->q;
    p.out = d->out;
    p.lse = d->lse;
    p.q_row = d->q_row_stride;
    p.out_row = d->out_row_stride;
    p.q_heads = d->q_heads;
    p.group = d->q_heads / kv->kv_heads;
    p.window = d->window;
    p.scale_log2 = scale_log2;
    unsigned char* ws = static_cast<unsigned char*>(d->workspace);
    p.tickets = reinterpret_cast<unsigned int*>(ws);
    p.part_ml = reinterpret_cast<float*>(ws + l.ml);
    p.part_o = reinterpret_cast<float*>(ws + l.o);
    const uint32_t limit = wait_kclocks.load(std::memory_order_relaxed);
    p.wait_clocks = limit != 0 ? static_cast<long long>(limit) << 10 : kWaitClocks;
    // Few (row, head) pairs per KV head stream, many go to tensor memory.  Measured at 2055-2900 keys, 32 / 8 heads, caches
    // larger than L2 (streaming : tensor memory, us):
    //                            16 sequences    8 sequences    2 sequences
    //   bf16, D = 128, 16 pairs    37 :  54        26 : 39        17 : 17
    //                  28 pairs    48 :  54        34 : 40        24 : 18
    //                  48 pairs    73 :  54        49 : 40        24 : 20
    //         D =  64, 16 pairs    26 :  35        19 : 26        12 : 15
    //                  28 pairs    32 :  35        24 : 26        16 : 15
    //                  48 pairs    51 :  36        34 : 26        17 : 16
    //   f32,  D = 128, 28 pairs    69 :  93        45 : 63        19 : 27
    //                  48 pairs    99 :  94        63 : 64        23 : 29
    //                  64 pairs   126 :  95        76 : 65        26 : 30
    //         D =  64, 28 pairs    46 :  55        30 : 37        14 : 19
    //                  48 pairs    64 :  56        40 : 38        16 : 19
    //                  64 pairs    82 :  56        50 : 38        18 : 20
    // Between 17 and 32 pairs of 16-bit rows what counts is how many CTAs share a cell, since the streaming kernel's joins
    // are the slower ones: it takes them when there is a cell (sequence and KV head) for two of three multiprocessors (the
    // border lies somewhere below the 64 cells of 8 sequences, above the 16 of two).
    const uint64_t pairs = static_cast<uint64_t>(d->max_rows < batch->total_rows ? d->max_rows : batch->total_rows) * p.group;
    const uint32_t narrow = stream_pairs(d->dtype);
    const bool many_cells = static_cast<uint64_t>(batch->n_seqs) * kv->kv_heads * 3 >= sms * 2ull;
    const uint64_t streams = d->dtype == ITK_ROW_F32 ? 48 : many_cells ? 32 : 16;
    const cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    const cudaError_t err = pairs > streams && tc_takes(p.pool) ? launch_tc(p, d->dtype, sms, s)
                                                                : launch_stream(p, d->dtype, pairs > narrow, sms, s);
    return err == cudaSuccess ? 0 : e.cuda("paged attention launch failed", err);
}
