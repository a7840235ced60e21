// Appending keys and values to the paged 8-bit cache, with the rotation of
// queries and keys on the way, and reading tokens back as rows.
#include "gemm.cuh"
#include "kvcache.cuh"

namespace ditch {
namespace kv {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kTile = 16;    // tokens of a block that one warp holds
constexpr int kQPasses = 2;  // query rows a lane group rotates one after another

// ---- eight consecutive dimensions of a row --------------------------------------
__device__ __forceinline__ void unpack2(uint32_t u, int dtype, float &a, float &b) {
    if (dtype == kBf16) {
        a = __uint_as_float(u << 16);
        b = __uint_as_float(u & 0xffff0000u);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<__half2 *>(&u));
        a = f.x;
        b = f.y;
    }
}

__device__ __forceinline__ void load8(const Rows &r, long long at, float (&x)[8]) {
    if (!r.vec) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = load1(r, at + i);
    } else if (r.dtype == kF32) {
        const float4 *s = reinterpret_cast<const float4 *>(static_cast<const float *>(r.p) + at);
        const float4 a = s[0], b = s[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(r.p) + at);
        unpack2(u.x, r.dtype, x[0], x[1]);
        unpack2(u.y, r.dtype, x[2], x[3]);
        unpack2(u.z, r.dtype, x[4], x[5]);
        unpack2(u.w, r.dtype, x[6], x[7]);
    }
}

__device__ __forceinline__ uint32_t pack2(int dtype, float a, float b) {
    if (dtype == kBf16) return f32_to_bf16_bits(a) | static_cast<uint32_t>(f32_to_bf16_bits(b)) << 16;
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ void store8(const Rows &r, long long at, const float (&x)[8]) {
    if (!r.vec) {
#pragma unroll
        for (int i = 0; i < 8; i++) store1(r, at + i, x[i]);
    } else if (r.dtype == kF32) {
        float4 *d = reinterpret_cast<float4 *>(static_cast<float *>(r.p) + at);
        d[0] = make_float4(x[0], x[1], x[2], x[3]);
        d[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(r.p) + at) =
            make_uint4(pack2(r.dtype, x[0], x[1]), pack2(r.dtype, x[2], x[3]), pack2(r.dtype, x[4], x[5]),
                       pack2(r.dtype, x[6], x[7]));
    }
}

// A head is held by LPT lanes, 16 dimensions each: two runs of 8. In the
// rotated part the runs are the two halves of eight pairs (neox) or the
// pairs' neighbours (gptj); either way lane l has pairs 8 l .. 8 l + 7.
struct Part {
    int c0, c1;  // first dimension of each run
    bool on, turns;
};

__device__ __forceinline__ Part part_of(int l, int dim, const Rope &r, bool rotate) {
    Part p;
    const int h8 = r.half >> 3;
    p.on = 16 * l < dim;
    p.turns = rotate && l < h8;
    const bool halves = r.style == 0 && rotate;
    p.c0 = p.turns && halves ? 8 * l : 16 * l;
    p.c1 = p.turns && halves ? 8 * l + r.half : 16 * l + 8;
    return p;
}

// The products and their sums are rounded one by one (no fused multiply-add),
// so that the codes are those of the formula in f32, bit for bit.
__device__ __forceinline__ void turn(float &a, float &b, float c, float s) {
    const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
    a = x;
}

__device__ __forceinline__ void rotate16(const Rope &r, int l, int pos, float (&x0)[8], float (&x1)[8]) {
    const long long at = static_cast<long long>(pos) * r.half + 8 * l;
    const float4 *ct = reinterpret_cast<const float4 *>(r.cos_t + at);
    const float4 *st = reinterpret_cast<const float4 *>(r.sin_t + at);
    const float4 c0 = __ldg(ct), c1 = __ldg(ct + 1), s0 = __ldg(st), s1 = __ldg(st + 1);
    const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    const float s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
    if (r.style == 0) {
#pragma unroll
        for (int i = 0; i < 8; i++) turn(x0[i], x1[i], c[i], s[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            turn(x0[2 * i], x0[2 * i + 1], c[i], s[i]);
            turn(x1[2 * i], x1[2 * i + 1], c[4 + i], s[4 + i]);
        }
    }
}

// ---- codes ---------------------------------------------------------------------------
// Two values (already divided by the scale) to two E4M3 codes, a in the low byte.
__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}

// Round to nearest even and clamp to -127..127; a NaN gives 0.
__device__ __forceinline__ uint32_t int8_code(float v) {
    return static_cast<uint32_t>(max(-127, min(127, __float2int_rn(v)))) & 0xff;
}

__device__ __forceinline__ uint32_t encode4(bool fp8, const float *x, float f) {
    if (fp8) return e4m3_pair(x[0] * f, x[1] * f) | e4m3_pair(x[2] * f, x[3] * f) << 16;
    return int8_code(x[0] * f) | int8_code(x[1] * f) << 8 | int8_code(x[2] * f) << 16 | int8_code(x[3] * f) << 24;
}

__device__ __forceinline__ uint2 encode8(bool fp8, const float (&x)[8], float f) {
    return make_uint2(encode4(fp8, x, f), encode4(fp8, x + 4, f));
}

// ---- append --------------------------------------------------------------------------
// The last sequence whose first slot is at most `slot`. Sequences of any
// lengths get enough slots for their blocks when sequence s starts at slot
// offsets[s] / block + 2 s (n new tokens reach at most n / block + 2 blocks).
__device__ __forceinline__ int seq_of_slot(const Batch &b, int block_shift, int slot) {
    int lo = 0, hi = b.n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((__ldg(b.offsets + mid) >> block_shift) + 2 * mid <= slot) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ int seq_of_row(const Batch &b, int row) {
    // one new token each: the row is the sequence
    if (row < b.n_seqs && __ldg(b.offsets + row) == row && __ldg(b.offsets + row + 1) == row + 1) return row;
    int lo = 0, hi = b.n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (__ldg(b.offsets + mid) <= row) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Bound by HBM (rows in, rotated queries and codes out) once there are more
// than a few thousand tokens, by latency below. One CTA is four warps; a warp
// holds 16 tokens of one scale's block for one kv head (of keys or of
// values) in registers, so a block of 16 / 32 / 64 tokens takes 1 / 2 / 4
// warps and every row is read once: the magnitudes meet by warp reduction
// and shared memory, then the same registers are rounded to codes. The CTAs
// after those of keys and values rotate the query rows.
template <int LPT>
__global__ void __launch_bounds__(kThreads) k_kv_append(AppendParams p, int kv_ctas, int ctas_per_slot) {
    constexpr int kTpp = 32 / LPT;           // tokens of a pass
    constexpr int kPasses = kTile / kTpp;
    __shared__ uint32_t s_top[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane & (LPT - 1), sub = lane / LPT;
    const Batch &b = p.b;
    const bool rope = p.r.cos_t != nullptr;

    if (static_cast<int>(blockIdx.x) >= kv_ctas) {  // query rows
        const Part part = part_of(l, p.c.dim, p.r, rope);
        const long long rows = static_cast<long long>(b.n_tokens) * p.q.heads;
        long long row = (static_cast<long long>(blockIdx.x - kv_ctas) * kWarps + warp) * (kTpp * kQPasses) + sub;
        int seq = -1;
#pragma unroll
        for (int it = 0; it < kQPasses; it++, row += kTpp) {
            if (row >= rows || !part.on) break;
            const int tok = static_cast<int>(row / p.q.heads), head = static_cast<int>(row - static_cast<long long>(tok) * p.q.heads);
            const long long at = tok * p.q.ts + head * p.q.hs, to = tok * p.qo.ts + head * p.qo.hs;
            float x0[8], x1[8];
            load8(p.q, at + part.c0, x0);
            load8(p.q, at + part.c1, x1);
            if (part.turns) {
                if (seq < 0) seq = seq_of_row(b, tok);
                while (seq + 1 < b.n_seqs && __ldg(b.offsets + seq + 1) <= tok) seq++;
                const Span a = span_of(b, p.c.page_shift, seq, p.status);
                const int i = tok - a.row0;
                if (i < 0 || i >= a.n) continue;  // a bad offset: already flagged
                rotate16(p.r, l, a.len - a.n + i, x0, x1);
            }
            store8(p.qo, to + part.c0, x0);
            store8(p.qo, to + part.c1, x1);
        }
        return;
    }

    const int block = 1 << p.c.block_shift, wpu = block / kTile;  // warps of a unit
    const int slot = blockIdx.x / ctas_per_slot;
    const int unit = (blockIdx.x - slot * ctas_per_slot) * (kWarps / wpu) + warp / wpu;
    const int seq = b.max_new == 1 ? slot : seq_of_slot(b, p.c.block_shift, slot);
    const int nth = b.max_new == 1 ? 0 : slot - ((__ldg(b.offsets + seq) >> p.c.block_shift) + 2 * seq);
    const Span a = span_of(b, p.c.page_shift, seq, p.status);
    const int start = a.len - a.n;
    const int lo = ((start >> p.c.block_shift) + nth) << p.c.block_shift;  // first token of the block
    if (a.n == 0 || lo >= a.len) return;
    const bool live = unit < 2 * p.c.heads;
    const bool value = unit >= p.c.heads;
    const int head = value ? unit - p.c.heads : unit;
    const int page = page_of(p.c, b, seq, lo, p.status);
    const Rows &src = value ? p.v : p.k, &dst = value ? p.vo : p.ko;
    const Part part = part_of(l, p.c.dim, p.r, rope && !value);
    float *scale = live && page >= 0 ? (value ? p.c.vs : p.c.ks) + scale_at(p.c, page, head, lo) : nullptr;
    const uint32_t kept = scale && lo < start ? __float_as_uint(*scale) : 0u;  // scales are not negative

    const int t0 = lo + (warp & (wpu - 1)) * kTile + sub;  // this lane's first token
    float x0[kPasses][8], x1[kPasses][8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kPasses; i++) {
        const int t = t0 + i * kTpp;
        if (live && part.on && t >= start && t < a.len) {
            const long long tok = a.row0 + (t - start), at = tok * src.ts + head * src.hs;
            load8(src, at + part.c0, x0[i]);
            load8(src, at + part.c1, x1[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < kPasses; i++) {
        const int t = t0 + i * kTpp;
        if (live && part.on && t >= start && t < a.len) {
            if (part.turns) rotate16(p.r, l, t, x0[i], x1[i]);
            // magnitudes as bits: an infinity is above every number, a NaN above that
#pragma unroll
            for (int j = 0; j < 8; j++)
                top = max(top, max(__float_as_uint(x0[i][j]) & 0x7fffffffu, __float_as_uint(x1[i][j]) & 0x7fffffffu));
            if (dst.p) {
                const long long to = (a.row0 + (t - start)) * dst.ts + head * dst.hs;
                store8(dst, to + part.c0, x0[i]);
                store8(dst, to + part.c1, x1[i]);
            }
        }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (wpu > 1) {
        if (lane == 0) s_top[warp] = top;
        __syncthreads();
        const int first = warp & ~(wpu - 1);
        for (int w = 0; w < wpu; w++) top = max(top, s_top[first + w]);
    }
    if (!scale) return;

    float fresh = __fdiv_rn(__uint_as_float(top), p.c.fp8 ? 448.0f : 127.0f);
    if (top >= 0x7f800000u) fresh = __uint_as_float(0x7fc00000u);
    else if (fresh < 1.17549435e-38f) fresh = 0.0f;
    const uint32_t s_bits = max(kept, __float_as_uint(fresh));
    const float s = __uint_as_float(s_bits);
    const bool nil = s == 0.0f || s_bits >= 0x7f800000u;
    const float inv = nil ? 0.0f : __fdiv_rn(1.0f, s);
    const bool again = kept != 0 && s_bits > kept;  // earlier tokens of the block get the new scale
    const float ratio = nil ? 0.0f : __fdiv_rn(__uint_as_float(kept), s);
    uint8_t *codes = (value ? p.c.v : p.c.k) + code_at(p.c, page, head, lo);
#pragma unroll
    for (int i = 0; i < kPasses; i++) {
        const int t = t0 + i * kTpp;
        if (!part.on || t >= a.len) continue;
        uint8_t *row = codes + static_cast<long long>(t - lo) * p.c.dim;
        uint2 *r0 = reinterpret_cast<uint2 *>(row + part.c0), *r1 = reinterpret_cast<uint2 *>(row + part.c1);
        if (t < start) {
            if (!again) continue;
            const uint2 u0 = *r0, u1 = *r1;
            decode4(p.c.fp8, u0.x, x0[i]);
            decode4(p.c.fp8, u0.y, x0[i] + 4);
            decode4(p.c.fp8, u1.x, x1[i]);
            decode4(p.c.fp8, u1.y, x1[i] + 4);
        }
        const float f = t < start ? ratio : inv;
        uint2 e0 = make_uint2(0, 0), e1 = make_uint2(0, 0);
        if (!nil) {
            e0 = encode8(p.c.fp8, x0[i], f);
            e1 = encode8(p.c.fp8, x1[i], f);
        }
        *r0 = e0;
        *r1 = e1;
    }
    if ((warp & (wpu - 1)) == 0 && lane == 0) *scale = s;
}

// ---- read ------------------------------------------------------------------------------
// Bound by HBM. A thread turns 16 codes (one 16-byte load) of one token and
// head into 16 values; keys, then values.
__global__ void __launch_bounds__(256) k_kv_read(ReadParams p) {
    const int parts = p.c.dim >> 4;
    const long long per = static_cast<long long>(p.b.n_tokens) * p.c.heads * parts;
    long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= 2 * per) return;
    const bool value = i >= per;
    if (value) i -= per;
    const long long row = i / parts;
    const int d = static_cast<int>(i - row * parts) * 16;
    const int tok = static_cast<int>(row / p.c.heads), head = static_cast<int>(row - static_cast<long long>(tok) * p.c.heads);
    const int seq = seq_of_row(p.b, tok);
    const Span a = span_of(p.b, p.c.page_shift, seq, p.status);
    const int k = tok - a.row0;
    if (k < 0 || k >= a.n) return;
    const int t = a.len - a.n + k;
    const int page = page_of(p.c, p.b, seq, t, p.status);
    if (page < 0) return;
    const uint4 u = *reinterpret_cast<const uint4 *>((value ? p.c.v : p.c.k) + code_at(p.c, page, head, t) + d);
    const float s = (value ? p.c.vs : p.c.ks)[scale_at(p.c, page, head, t)];
    float x[8], y[8];
    decode4(p.c.fp8, u.x, x);
    decode4(p.c.fp8, u.y, x + 4);
    decode4(p.c.fp8, u.z, y);
    decode4(p.c.fp8, u.w, y + 4);
#pragma unroll
    for (int j = 0; j < 8; j++) {
        x[j] *= s;
        y[j] *= s;
    }
    const Rows &o = value ? p.vo : p.ko;
    const long long at = tok * o.ts + head * o.hs + d;
    store8(o, at, x);
    store8(o, at + 8, y);
}

}  // namespace

bool codes_map(CUtensorMap *map, const Cache &c, const void *codes, int row_bytes, int tokens) {
    const cuuint64_t page = (cuuint64_t)c.heads << c.page_shift;
    const cuuint64_t dims[3] = {(cuuint64_t)c.dim, page, (cuuint64_t)c.n_pages};
    const cuuint64_t strides[2] = {(cuuint64_t)c.dim, page * c.dim};
    const cuuint32_t box[3] = {(cuuint32_t)row_bytes, (cuuint32_t)tokens, 1};
    return tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, codes, dims, strides, box,
                      row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

cudaError_t append(const AppendParams &p, cudaStream_t s) {
    const int lpt = p.c.dim <= 32 ? 2 : p.c.dim <= 64 ? 4 : 8;
    const int block = 1 << p.c.block_shift, units = kWarps / (block / kTile);
    const long long slots = p.b.max_new == 1 ? p.b.n_seqs : (long long)(p.b.n_tokens / block) + 2LL * p.b.n_seqs;
    const int per_slot = (2 * p.c.heads + units - 1) / units;
    const long long kv_ctas = slots * per_slot;
    const long long rows_per_cta = (long long)kWarps * (32 / lpt) * kQPasses;
    const long long q_ctas = p.q.p ? ((long long)p.b.n_tokens * p.q.heads + rows_per_cta - 1) / rows_per_cta : 0;
    if (kv_ctas + q_ctas > 0x7fffffffLL) return cudaErrorInvalidValue;
    const unsigned grid = (unsigned)(kv_ctas + q_ctas);
    if (lpt == 2) k_kv_append<2><<<grid, kThreads, 0, s>>>(p, (int)kv_ctas, per_slot);
    else if (lpt == 4) k_kv_append<4><<<grid, kThreads, 0, s>>>(p, (int)kv_ctas, per_slot);
    else k_kv_append<8><<<grid, kThreads, 0, s>>>(p, (int)kv_ctas, per_slot);
    return cudaGetLastError();
}

cudaError_t read_back(const ReadParams &p, cudaStream_t s) {
    const long long n = 2LL * p.b.n_tokens * p.c.heads * (p.c.dim / 16);
    const long long ctas = (n + 255) / 256;
    if (ctas > 0x7fffffffLL) return cudaErrorInvalidValue;
    k_kv_read<<<(unsigned)ctas, 256, 0, s>>>(p);
    return cudaGetLastError();
}

}  // namespace kv
}  // namespace ditch
