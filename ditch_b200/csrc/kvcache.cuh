// The paged 8-bit key / value cache and the attentions over it and over
// contiguous rows (include/ditch_cuda.h): launch parameters and the device
// helpers that their kernels share.
#pragma once

#include <atomic>

#include "common.cuh"

namespace ditch {
namespace kv {

enum RowType : int { kF32 = 0, kF16 = 1, kBf16 = 2 };  // DITCH_DTYPE_F32 / F16 / BF16

// Rows [tokens][heads][head_dim]; vec: every head is 16-byte aligned.
struct Rows {
    void *p;
    long long ts, hs;
    int dtype, heads, vec;
};

struct Cache {
    uint8_t *k, *v;
    float *ks, *vs;
    long long n_pages;
    int fp8, heads, dim;
    int page_shift, block_shift;  // log2 of the tokens of a page and of a scale's block
};

struct Batch {
    const int32_t *offsets, *lens, *pages;
    int n_seqs, n_tokens, max_new, max_len, max_pages;
};

struct Rope {
    const float *cos_t, *sin_t;
    int len, half, style;
};

struct AppendParams {
    Cache c;
    Batch b;
    Rope r;
    Rows q, qo, k, v, ko, vo;  // q.p, ko.p and vo.p may be null
    int *status;
};

struct ReadParams {
    Cache c;
    Batch b;
    Rows ko, vo;
    int *status;
};

struct AttendParams {
    Cache c;
    Batch b;
    Rows q, out;
    float scale;
    int window, sinks;  // window 0: every earlier token
    void *ws;
    int *status;
};

struct Ragged {
    const int32_t *qo, *ko;
    int n_seqs, n_q, n_kv, max_q, max_kv;
};

struct WindowParams {
    Ragged b;
    Rows q, k, v, out;
    int dim;
    float scale;
    int window, sinks;
    int *status;
};

// The tensor map of a pool's K or V codes for boxes of `tokens` tokens of one
// page and head: rows of row_bytes (64 or 128) with as wide a swizzle, zeros
// past the head's dimensions. Coordinates (0, head * page_tokens + t, page).
bool codes_map(CUtensorMap *map, const Cache &c, const void *codes, int row_bytes, int tokens);

cudaError_t append(const AppendParams &p, cudaStream_t s);
cudaError_t read_back(const ReadParams &p, cudaStream_t s);
size_t attend_workspace(const Cache &c, const Batch &b, int q_heads, int sms);
cudaError_t attend(const AttendParams &p, int sms, cudaStream_t s);
cudaError_t window_attention(const WindowParams &p, int sms, cudaStream_t s);
constexpr int kTiledSeqs = 65535;  // sequences that the tiled kernel takes (a grid dimension)
// The tiled (tcgen05) form of attend, for many rows; and what it costs.
cudaError_t attend_tiled(const AttendParams &p, cudaStream_t s);
double tiled_rounds(const AttendParams &p, int sms, long long seen);

// Raises a kernel's dynamic shared memory limit on the current device, once
// for each device.
struct SmemOptIn {
    std::atomic<uint64_t> done{0};
    cudaError_t set(const void *kernel, int bytes) {
        int d = 0;
        cudaError_t e = cudaGetDevice(&d);
        if (e != cudaSuccess || d > 63 || (done.load(std::memory_order_acquire) >> d & 1) == 0) {
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
            if (e == cudaSuccess && d <= 63) done.fetch_or(1ull << d, std::memory_order_release);
        }
        return e;
    }
};

// ---- a sequence of a batch ---------------------------------------------------
// Rows [row0, row0 + n) of the call are the last n of `len` tokens.
struct Span {
    int row0, n, len;
};

__device__ __forceinline__ void flag(int *status) {
    if (status) atomicExch(status, kKernelBadArgument);
}

// Sequence s of the batch; n = 0 (and the status word set) when the device's
// numbers leave the host's bounds.
__device__ __forceinline__ Span span_of(const Batch &b, int page_shift, int s, int *status) {
    Span a;
    a.row0 = __ldg(b.offsets + s);
    const int end = __ldg(b.offsets + s + 1);
    a.len = __ldg(b.lens + s);
    a.n = end - a.row0;
    const bool ok = a.row0 >= 0 && end <= b.n_tokens && a.n >= 0 && a.n <= b.max_new && a.len >= a.n &&
                    a.len <= b.max_len && a.len <= (static_cast<long long>(b.max_pages) << page_shift);
    if (!ok) {
        flag(status);
        a.n = a.len = 0;
    }
    return a;
}

// The page of token t of sequence s, or -1 (and the status word set).
__device__ __forceinline__ int page_of(const Cache &c, const Batch &b, int s, int t, int *status) {
    const int page = __ldg(b.pages + static_cast<long long>(s) * b.max_pages + (t >> c.page_shift));
    if (page >= 0 && page < c.n_pages) return page;
    flag(status);
    return -1;
}

// Byte offset of token t's codes within the pool, and index of its scale.
__device__ __forceinline__ long long code_at(const Cache &c, int page, int head, int t) {
    const long long row = ((static_cast<long long>(page) * c.heads + head) << c.page_shift) + (t & ((1 << c.page_shift) - 1));
    return row * c.dim;
}

__device__ __forceinline__ long long scale_at(const Cache &c, int page, int head, int t) {
    const int in_page = t & ((1 << c.page_shift) - 1);
    return ((static_cast<long long>(page) * c.heads + head) << (c.page_shift - c.block_shift)) + (in_page >> c.block_shift);
}

// ---- codes -----------------------------------------------------------------------
// Four codes' values without their scale.
__device__ __forceinline__ void decode4(bool fp8, uint32_t u, float *x) {
    if (fp8) {
        const float2 a = e4m3x2_f32(u & 0xffff), b = e4m3x2_f32(u >> 16);
        x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = static_cast<float>(static_cast<int8_t>(u >> (8 * i)));
    }
}

// ---- rows -----------------------------------------------------------------------
__device__ __forceinline__ float load1(const Rows &r, long long at) {
    if (r.dtype == kF32) return static_cast<const float *>(r.p)[at];
    const uint16_t u = static_cast<const uint16_t *>(r.p)[at];
    return r.dtype == kBf16 ? bf16_bits_to_f32(u) : __half2float(__ushort_as_half(u));
}

__device__ __forceinline__ void store1(const Rows &r, long long at, float v) {
    if (r.dtype == kF32) static_cast<float *>(r.p)[at] = v;
    else if (r.dtype == kBf16) static_cast<uint16_t *>(r.p)[at] = f32_to_bf16_bits(v);
    else static_cast<__half *>(r.p)[at] = __float2half_rn(v);
}

// Four values of a row, at a multiple of four.
__device__ __forceinline__ float4 load4(const Rows &r, long long at) {
    if (!r.vec) return make_float4(load1(r, at), load1(r, at + 1), load1(r, at + 2), load1(r, at + 3));
    if (r.dtype == kF32) return *reinterpret_cast<const float4 *>(static_cast<const float *>(r.p) + at);
    const uint2 u = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(r.p) + at);
    if (r.dtype == kBf16)
        return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                           __uint_as_float(u.y & 0xffff0000u));
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
}

// Four values to a 16-byte aligned row, at a multiple of four.
__device__ __forceinline__ void store4(const Rows &r, long long at, float4 v) {
    if (r.dtype == kF32) {
        *reinterpret_cast<float4 *>(static_cast<float *>(r.p) + at) = v;
    } else if (r.dtype == kBf16) {
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(r.p) + at) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
    } else {
        const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(r.p) + at) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
}

}  // namespace kv
}  // namespace ditch
