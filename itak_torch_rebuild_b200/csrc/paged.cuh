// What the paged-cache kernels share: element types of rows and pages, the batch as a launch sees it, and the host
// side's refusals.
//
// Pages:  element (page, head, row, channel) at page * page_stride + head * head_stride + row * row_stride + channel;
//         the key of position p of sequence s is row p % page_size of page table[s][p / page_size].
// Batch:  sequence s owns the packed rows [row_start[s], row_start[s + 1]) and kv_len[s] keys, its new rows included,
//         so that its row i sits at position kv_len[s] - rows + i.  These arrays are read on the device only; whatever
//         they hold, no kernel follows a page number outside the pool or a row outside the packed tensors.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include <atomic>

#include "../../include/itak_cuda_compute.h"
#include "kv_convert.cuh"

namespace itk {
namespace paged {

constexpr uint32_t kMaxSeqs = 1024;
constexpr uint32_t kMaxHeadDim = 256;
constexpr uint32_t kMaxLen = 1u << 30;  // keys of one sequence
constexpr uint32_t kMaxStated = 0x7fffffffu;  // stated lengths count as this at most

// Bits of itk_paged_batch::status.
constexpr uint32_t kBadPage = 1u, kLongSeq = 2u, kBeforeStart = 4u, kBadStarts = 8u, kWaitRanOut = 16u;

struct Pool {
    void* k;
    void* v;
    uint64_t page_stride, head_stride, row_stride;  // elements
    uint32_t n_pages, page_shift;                   // page_size = 1 << page_shift
    uint32_t kv_heads, head_dim;
};

struct Batch {
    const uint32_t* table;
    const uint32_t* row_start;
    const uint32_t* kv_len;
    uint32_t* status;
    uint32_t n_seqs, table_width, table_stride, total_rows;
};

__device__ __forceinline__ void raise(const Batch& b, uint32_t bits) {
    if (b.status) atomicOr(b.status, bits);
}

// Keys that a row of the table has places for.
__device__ __forceinline__ uint32_t room_of(const Batch& b, uint32_t page_shift) {
    return static_cast<uint32_t>(min(static_cast<uint64_t>(b.table_width) << page_shift, static_cast<uint64_t>(kMaxLen)));
}

// One sequence of the batch, with the rows that the packed tensors do not hold cut off (see itk_paged_batch for what is
// reported).  Positions go by the stated length, whatever the table has room for: rows that moved to fit would lie over
// keys that live there.  Of its keys there are min(len, room).
struct Seq {
    uint32_t row0, rows;  // packed rows
    uint32_t len;         // stated keys
    int32_t pos0;         // position of the first row; negative when the new rows reach before position 0
};
__device__ __forceinline__ Seq seq_of(const Batch& b, uint32_t s, uint32_t page_shift) {
    const uint32_t lo = b.row_start[s], hi = b.row_start[s + 1];
    const uint32_t stated = b.kv_len[s];
    const uint32_t room = room_of(b, page_shift);
    Seq q;
    q.row0 = min(lo, b.total_rows);
    const uint32_t end = min(hi, b.total_rows);
    q.rows = end > q.row0 ? end - q.row0 : 0u;
    q.len = min(stated, kMaxStated);
    q.pos0 = static_cast<int32_t>(q.len) - static_cast<int32_t>(q.rows);
    uint32_t bits = 0;
    if (hi < lo || hi > b.total_rows) bits |= kBadStarts;
    if (stated > room) bits |= kLongSeq;
    if (q.pos0 < 0) bits |= kBeforeStart;
    if (bits) raise(b, bits);
    return q;
}

// Softmax weights are kept 2^kLift times larger than 2^(c s - m) where they are rounded to halfs: with a running maximum that lags
// by up to 2^8 they reach 2^15, and small ones stay clear of the type's subnormal steps - 2^-32 of the row's largest instead of
// 2^-25, which over 2^15 keys under one that outshines them would add up to 1e-3 of a result.  The sum scales alike, and
// is scaled back for the log-sum-exp.  bf16 has the range of f32 and needs none.
template <typename P>
constexpr float kLift = 0.f;
template <>
constexpr float kLift<__half> = 7.f;
template <typename P>
constexpr float kUnlift = 1.f;
template <>
constexpr float kUnlift<__half> = 1.f / 128.f;

// What an attention launch gets (both kernels).
struct AttnParams {
    Pool pool;
    Batch batch;
    const void* q;
    void* out;
    float* lse;
    uint64_t q_row, out_row;  // elements
    int device;
    uint32_t q_heads, group, window;
    float scale_log2;  // scale * log2(e)
    unsigned int* tickets;  // zero between launches
    float* part_ml;         // [part][row][2]: running maximum (log2 domain) and sum
    float* part_o;          // [part][row][D]: unnormalised outputs
    long long wait_clocks;  // bound of the tensor-memory kernel's waits, SM clocks
};

// Takes a ticket: orders the block's stores before it (all of them precede a barrier that the caller has passed) and what
// the block reads behind a further barrier after it, with one instruction of one thread.
__device__ __forceinline__ uint32_t take_ticket(unsigned int* counter) {
    uint32_t ticket;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;\n" : "=r"(ticket) : "l"(counter) : "memory");
    return ticket;
}

// ---- element types ------------------------------------------------------------------------------------------------

// Eight consecutive channels of a row as they travel: two 16-byte words of f32, one of a 16-bit type.
template <typename T>
struct Vec8;
template <>
struct Vec8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = reinterpret_cast<const float4*>(p)[0];
        b = reinterpret_cast<const float4*>(p)[1];
    }
    __device__ __forceinline__ void store(float* p) const {
        reinterpret_cast<float4*>(p)[0] = a;
        reinterpret_cast<float4*>(p)[1] = b;
    }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    }
    __device__ __forceinline__ void set(const float (&f)[8]) {
        a = make_float4(f[0], f[1], f[2], f[3]);
        b = make_float4(f[4], f[5], f[6], f[7]);
    }
};
template <>
struct Vec8<__half> {
    uint4 w;
    __device__ __forceinline__ void load(const __half* p) { w = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void store(__half* p) const { *reinterpret_cast<uint4*>(p) = w; }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __half2float(__ushort_as_half(static_cast<unsigned short>(u[i] & 0xffffu)));
            f[2 * i + 1] = __half2float(__ushort_as_half(static_cast<unsigned short>(u[i] >> 16)));
        }
    }
    __device__ __forceinline__ void set(const float (&f)[8]) {
        w = pack8(make_float4(f[0], f[1], f[2], f[3]), make_float4(f[4], f[5], f[6], f[7]));
    }
};
template <>
struct Vec8<__nv_bfloat16> {
    uint4 w;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { w = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = w; }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(u[i] << 16);
            f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
    __device__ __forceinline__ void set(const float (&f)[8]) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
        w = make_uint4(u[0], u[1], u[2], u[3]);
    }
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __ushort_as_half(f32_to_f16_bits(x)); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// The kernels are launched as programmatic dependents: their blocks take their places while the kernel before them in the
// stream still runs, and wait here before they touch memory (2 us of a call that follows another).
// What a predecessor may have written - the table, starts, lengths, rows - is read with plain loads: the path for data that is
// read-only while a kernel runs is not for them, since this kernel runs while they are written.
__device__ __forceinline__ void after_predecessor() {
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
}

// ---- host side ------------------------------------------------------------------------------------------------------

// Writes the reason of a refusal into the caller's buffer.
struct ErrorText {
    char* text;
    size_t len;
    ErrorText(char* t, size_t n) : text(t), len(n) {
        if (text && len) text[0] = '\0';
    }
    int refuse(int code, const char* fmt, unsigned long long a = 0, unsigned long long b = 0) const {
        if (text && len) snprintf(text, len, fmt, a, b);
        return code;
    }
    int invalid(const char* fmt, unsigned long long a = 0, unsigned long long b = 0) const {
        return refuse(ITK_ERR_INVALID_ARGUMENT, fmt, a, b);
    }
    int cuda(const char* what, cudaError_t e) const {
        if (text && len) snprintf(text, len, "%s: %s", what, cudaGetErrorString(e));
        return ITK_ERR_CUDA;
    }
};

// An error that is reported to the caller is not left pending in the thread as well, where a later call would take it for
// its own: a launch that ran must not be reported as one that failed, or its caller may rotate rows in place twice.
inline cudaError_t handled(cudaError_t e) {
    if (e != cudaSuccess) cudaGetLastError();
    return e;
}

// Makes `device` current for the call and puts the caller's back.
class DeviceScope {
public:
    explicit DeviceScope(int device) {
        err = handled(cudaGetDevice(&prev_));
        if (err == cudaSuccess && prev_ != device) {
            err = handled(cudaSetDevice(device));
            changed_ = err == cudaSuccess;
        }
    }
    ~DeviceScope() {
        if (changed_) cudaSetDevice(prev_);
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
    cudaError_t err = cudaSuccess;

private:
    int prev_ = 0;
    bool changed_ = false;
};

// Whether something that holds for a device from its first use on (a kernel's shared-memory limit) has been done there.
// Two threads may both find it undone and do it twice.
class OncePerDevice {
public:
    bool done(int device) const { return device >= 0 && device < 64 && ((bits_.load(std::memory_order_acquire) >> device) & 1u) != 0; }
    void mark(int device) {
        if (device >= 0 && device < 64) bits_.fetch_or(1ull << device, std::memory_order_release);
    }

private:
    std::atomic<uint64_t> bits_{0};
};

// The launch's own result, whatever was pending before it.
template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), uint32_t grid, uint32_t threads, size_t smem, cudaStream_t s, const Args&... args) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return handled(cudaLaunchKernelEx(&cfg, kernel, args...));
}

constexpr uint64_t kMaxStride = 1ull << 38;

inline bool aligned_to(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Refusals that append and attention share; 0 when the pools and the batch can be used.
int check_pool(const itk_paged_kv* kv, const ErrorText& e, Pool* out);
int check_batch(const itk_paged_batch* b, const ErrorText& e, Batch* out);
int check_row_dtype(int32_t rows, int32_t pages, const ErrorText& e);

// The streaming kernel (any shape) on a device of `sms` multiprocessors.
constexpr uint32_t kStreamRows = 32;  // rows of one of its parts
inline uint32_t stream_ctas(uint32_t sms, uint32_t head_dim) { return head_dim <= 128 ? 2 * sms : sms; }
uint32_t stream_pairs(int32_t row_dtype);  // (row, head) pairs of its narrow block; the wide one has twice as many
cudaError_t launch_stream(const AttnParams& p, int32_t row_dtype, bool wide, uint32_t sms, cudaStream_t s);
// The tensor-memory kernel, for pools that it takes: head_dim up to 128, pages of at least 8 rows.
constexpr uint32_t kTcRows = 256, kTcWidth = 128;  // rows and channels of one of its parts
bool tc_takes(const Pool& pool);
cudaError_t launch_tc(const AttnParams& p, int32_t row_dtype, uint32_t sms, cudaStream_t s);

}  // namespace paged
}  // namespace itk
