// Appending keys and values to the paged 8-bit cache, with the rotation of
// queries and keys on the way, and reading tokens back as rows.
#include "gemm.cuh"
#include "kvcache.cuh"

namespace ditch {
namespace kv {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kQPasses = 2;  // query rows a lane group rotates, all loaded at once

// Tokens of a block that one warp holds when a head takes LPT lanes.
template <int LPT>
constexpr int tile_tokens() {
    return LPT == 2 ? 16 : 8;
}

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
    if (dtype == kBf16) return pack_bf16x2(a, b);
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

// cos and sin of a lane's eight pairs at one position.
struct Angles {
    float4 c0, c1, s0, s1;
};

__device__ __forceinline__ Angles angles_of(const Rope &r, int l, int pos) {
    const long long at = static_cast<long long>(pos) * r.half + 8 * l;
    const float4 *ct = reinterpret_cast<const float4 *>(r.cos_t + at);
    const float4 *st = reinterpret_cast<const float4 *>(r.sin_t + at);
    return Angles{__ldg(ct), __ldg(ct + 1), __ldg(st), __ldg(st + 1)};
}

__device__ __forceinline__ void rotate16(const Angles &a, int style, float (&x0)[8], float (&x1)[8]) {
    const float c[8] = {a.c0.x, a.c0.y, a.c0.z, a.c0.w, a.c1.x, a.c1.y, a.c1.z, a.c1.w};
    const float s[8] = {a.s0.x, a.s0.y, a.s0.z, a.s0.w, a.s1.x, a.s1.y, a.s1.z, a.s1.w};
    if (style == 0) {
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
// The last of n numbers i for which `le` holds (it holds for 0, and up to
// some i), by the whole warp: 32 at a time, as every step waits for memory.
template <class F>
__device__ __forceinline__ int warp_search(int n, int lane, F &&le) {
    int lo = 0;
    while (n > 1) {
        const int step = (n + 31) / 32, i = lane * step;
        const uint32_t yes = __ballot_sync(0xffffffffu, i < n && le(lo + i));
        const int at = yes ? (31 - __clz(yes)) * step : 0;
        lo += at;
        n = min(step, n - at);
    }
    return lo;
}

// The last sequence whose first slot is at most `slot`. Sequences of any
// lengths get enough slots for their blocks when sequence s starts at slot
// offsets[s] / block + 2 s (n new tokens reach at most n / block + 2 blocks).
__device__ __forceinline__ int seq_of_slot(const Batch &b, int block_shift, int slot, int lane) {
    return warp_search(b.n_seqs, lane, [&](int s) { return (__ldg(b.offsets + s) >> block_shift) + 2 * s <= slot; });
}

__device__ __forceinline__ int seq_of_row(const Batch &b, int row, int lane) {
    // one new token each: the row is the sequence
    if (row < b.n_seqs && __ldg(b.offsets + row) == row && __ldg(b.offsets + row + 1) == row + 1) return row;
    return warp_search(b.n_seqs, lane, [&](int s) { return __ldg(b.offsets + s) <= row; });
}

// Rotates (and copies) kTpp * kQPasses heads of one token's queries.
template <int LPT>
__device__ __forceinline__ void query_rows(const AppendParams &p, unsigned unit, int parts, int lane) {
    constexpr int kTpp = 32 / LPT;
    const int l = lane & (LPT - 1), sub = lane / LPT;
    const Batch &b = p.b;
    const bool rope = p.r.cos_t != nullptr;
    const Part part = part_of(l, p.c.dim, p.r, rope);
    const unsigned tok = unit / parts;
    if (tok >= static_cast<unsigned>(b.n_tokens)) return;
    const int head0 = (unit - tok * parts) * (kTpp * kQPasses) + sub;
    const Rows &q = p.q, &qo = p.qo;
    float x0[kQPasses][8], x1[kQPasses][8];
#pragma unroll
    for (int i = 0; i < kQPasses; i++) {
        const int head = head0 + i * kTpp;
        if (head >= q.heads || !part.on) continue;
        const long long at = tok * q.ts + head * q.hs;
        load8(q, at + part.c0, x0[i]);
        load8(q, at + part.c1, x1[i]);
    }
    if (rope) {
        const int seq = seq_of_row(b, tok, lane);
        const Span a = span_of(b, p.c.page_shift, seq, p.status);
        const int i = static_cast<int>(tok) - a.row0;
        if (i < 0 || i >= a.n) return;  // a bad offset: already flagged
        if (part.turns) {
            const Angles angles = angles_of(p.r, l, a.len - a.n + i);
#pragma unroll
            for (int k = 0; k < kQPasses; k++) rotate16(angles, p.r.style, x0[k], x1[k]);
        }
    }
#pragma unroll
    for (int i = 0; i < kQPasses; i++) {
        const int head = head0 + i * kTpp;
        if (head >= q.heads || !part.on) continue;
        const long long to = tok * qo.ts + head * qo.hs;
        store8(qo, to + part.c0, x0[i]);
        store8(qo, to + part.c1, x1[i]);
    }
}

// A block's new scale from the largest magnitude (as bits) among its new
// values and the scale it keeps, and what follows.
struct Scale {
    float s, inv, ratio;  // ratio: old codes to new ones
    bool nil, again;      // codes are 0; earlier tokens' codes are rounded again
};

__device__ __forceinline__ Scale scale_of(uint32_t top, uint32_t kept, bool fp8) {
    Scale r;
    float fresh = __fdiv_rn(__uint_as_float(top), fp8 ? 448.0f : 127.0f);
    if (top >= 0x7f800000u) fresh = __uint_as_float(0x7fc00000u);
    else if (fresh < 1.17549435e-38f) fresh = 0.0f;
    const uint32_t bits = max(kept, __float_as_uint(fresh));
    r.s = __uint_as_float(bits);
    r.nil = r.s == 0.0f || bits >= 0x7f800000u;
    r.inv = r.nil ? 0.0f : __fdiv_rn(1.0f, r.s);
    r.again = kept != 0 && bits > kept;
    r.ratio = r.nil ? 0.0f : __fdiv_rn(__uint_as_float(kept), r.s);
    return r;
}

__device__ __forceinline__ void put_codes16(bool fp8, uint8_t *row, const Part &part, bool nil, const float (&x0)[8], const float (&x1)[8], float f) {
    const uint2 zero = make_uint2(0, 0);
    *reinterpret_cast<uint2 *>(row + part.c0) = nil ? zero : encode8(fp8, x0, f);
    *reinterpret_cast<uint2 *>(row + part.c1) = nil ? zero : encode8(fp8, x1, f);
}

__device__ __forceinline__ void get_codes16(bool fp8, const uint8_t *row, const Part &part, float (&x0)[8], float (&x1)[8]) {
    const uint2 u0 = *reinterpret_cast<const uint2 *>(row + part.c0), u1 = *reinterpret_cast<const uint2 *>(row + part.c1);
    decode4(fp8, u0.x, x0);
    decode4(fp8, u0.y, x0 + 4);
    decode4(fp8, u1.x, x1);
    decode4(fp8, u1.y, x1 + 4);
}

// One new token of each sequence: bound by latency. LPT lanes take a unit
// (sequence, kv head, keys or values): its row, the block's scale, the codes;
// only where the scale grows do they go over the block's earlier tokens (for
// the n-th token of a block once in n times). The general kernel would give
// each unit 2 to 8 warps (128 sequences of 8 heads, blocks of 32 tokens: 17.6
// us).
template <int LPT>
__global__ void __launch_bounds__(kThreads) k_kv_append_step(AppendParams p, int kv_ctas, int parts) {
    constexpr int kUnits = 32 / LPT;  // of a warp
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane & (LPT - 1);
    if (static_cast<int>(blockIdx.x) >= kv_ctas) {
        query_rows<LPT>(p, (blockIdx.x - kv_ctas) * kWarps + warp, parts, lane);
        return;
    }
    const Batch &b = p.b;
    const unsigned unit = (blockIdx.x * kWarps + warp) * kUnits + lane / LPT, heads = p.c.heads;
    const unsigned seq = unit / (2 * heads);
    const bool in = seq < static_cast<unsigned>(b.n_seqs);
    const unsigned which = unit - seq * (2 * heads);
    const bool value = which >= heads;
    const int head = value ? which - heads : which;
    Span a = {0, 0, 0};
    if (in) a = span_of(b, p.c.page_shift, seq, p.status);
    const bool live = a.n == 1;
    const int t = a.len - 1, lo = t >> p.c.block_shift << p.c.block_shift;
    const Part part = part_of(l, p.c.dim, p.r, p.r.cos_t != nullptr && !value);
    float x0[8], x1[8];
    uint32_t top = 0;
    if (live && part.on) {
        const Rows &src = value ? p.v : p.k, &dst = value ? p.vo : p.ko;
        const long long at = a.row0 * src.ts + head * src.hs;
        load8(src, at + part.c0, x0);
        load8(src, at + part.c1, x1);
        if (part.turns) rotate16(angles_of(p.r, l, t), p.r.style, x0, x1);
#pragma unroll
        for (int j = 0; j < 8; j++)
            top = max(top, max(__float_as_uint(x0[j]) & 0x7fffffffu, __float_as_uint(x1[j]) & 0x7fffffffu));
        if (dst.p) {
            const long long to = a.row0 * dst.ts + head * dst.hs;
            store8(dst, to + part.c0, x0);
            store8(dst, to + part.c1, x1);
        }
    }
#pragma unroll
    for (int o = 1; o < LPT; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const int page = live ? page_of(p.c, b, seq, t, p.status) : -1;
    float *scale = page >= 0 ? (value ? p.c.vs : p.c.ks) + scale_at(p.c, page, head, t) : nullptr;
    const uint32_t kept = scale && lo < t ? __float_as_uint(*scale) : 0u;
    __syncwarp();  // every lane has read the scale
    if (!scale || !part.on) return;
    const Scale s = scale_of(top, kept, p.c.fp8);
    uint8_t *row = (value ? p.c.v : p.c.k) + code_at(p.c, page, head, lo);
    put_codes16(p.c.fp8, row + (t - lo) * p.c.dim, part, s.nil, x0, x1, s.inv);
    if (s.again)
        for (int i = 0; i < t - lo; i++) {
            get_codes16(p.c.fp8, row + i * p.c.dim, part, x0, x1);
            put_codes16(p.c.fp8, row + i * p.c.dim, part, s.nil, x0, x1, s.ratio);
        }
    if (l == 0) *scale = s.s;
}

// Bound by HBM (rows in, rotated queries and codes out) once there are more
// than a few thousand tokens, by latency below. A warp holds 8 tokens (16 of
// heads of at most 32 dimensions) of one scale's block for one kv head, of
// keys or of values, in registers, so every row is read once: a block's
// magnitudes meet by warp reduction and shared memory, then the same
// registers are rounded to codes. How many warps are on an SM decides the
// time: 8192 tokens of 8 and 32 heads at f32 took 89 us at 16 tokens a warp
// (16 warps), 72 us at 8 tokens and 24 warps; with 32 warps, at the price of a
// few spills, the pass with its read is 2 % to 10 % shorter again. The CTAs
// after those of keys and values rotate the query rows, a warp a few heads of
// one token, whose angles are loaded once (a kernel of their own for them: 10
// us more). 8192 tokens and the read of what was stored: 87 us, 4.6 TB/s.
template <int LPT>
__global__ void __launch_bounds__(kThreads, 4) k_kv_append(AppendParams p, int kv_ctas, int ctas_per_slot, int parts) {
    constexpr int kTpp = 32 / LPT;           // tokens of a pass
    constexpr int kTile = tile_tokens<LPT>(), kPasses = kTile / kTpp;
    __shared__ uint32_t s_top[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane & (LPT - 1), sub = lane / LPT;
    const Batch &b = p.b;
    const bool rope = p.r.cos_t != nullptr;

    if (static_cast<int>(blockIdx.x) >= kv_ctas) {
        if (blockIdx.x == gridDim.x - 1) {  // a sequence whose offsets decrease may have no slot to be reported from
            for (int x = threadIdx.x; x < b.n_seqs; x += kThreads) span_of(b, p.c.page_shift, x, p.status);
            return;
        }
        query_rows<LPT>(p, (blockIdx.x - kv_ctas) * kWarps + warp, parts, lane);
        return;
    }

    const int block = 1 << p.c.block_shift, wpu = block / kTile;  // warps of a unit
    const int slot = blockIdx.x / ctas_per_slot;
    const int unit = (blockIdx.x - slot * ctas_per_slot) * (kWarps / wpu) + warp / wpu;
    const int seq = seq_of_slot(b, p.c.block_shift, slot, lane);
    const int nth = slot - ((__ldg(b.offsets + seq) >> p.c.block_shift) + 2 * seq);
    if (nth < 0) return;  // rows before the first sequence's
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
            if (part.turns) rotate16(angles_of(p.r, l, t), p.r.style, x0[i], x1[i]);
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

    const Scale s = scale_of(top, kept, p.c.fp8);
    uint8_t *codes = (value ? p.c.v : p.c.k) + code_at(p.c, page, head, lo);
#pragma unroll
    for (int i = 0; i < kPasses; i++) {
        const int t = t0 + i * kTpp;
        if (!part.on || t >= a.len || (t < start && !s.again)) continue;
        uint8_t *row = codes + static_cast<long long>(t - lo) * p.c.dim;
        if (t < start) get_codes16(p.c.fp8, row, part, x0[i], x1[i]);
        put_codes16(p.c.fp8, row, part, s.nil, x0[i], x1[i], t < start ? s.ratio : s.inv);
    }
    if ((warp & (wpu - 1)) == 0 && lane == 0) *scale = s.s;
}

// ---- read ------------------------------------------------------------------------------
// Bound by HBM. A warp takes one token, whose page is looked up once; a lane
// turns 16 codes (one 16-byte load) at a time into 16 values, keys and values
// of all heads. (A thread for each 16 codes, with its own lookups: 24.6 us
// for 8192 tokens of 8 heads.)
__global__ void __launch_bounds__(256) k_kv_read(ReadParams p) {
    const int tok = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (tok >= p.b.n_tokens) return;
    const int seq = seq_of_row(p.b, tok, lane);
    const Span a = span_of(p.b, p.c.page_shift, seq, p.status);
    const int k = tok - a.row0;
    if (k < 0 || k >= a.n) return;
    const int t = a.len - a.n + k;
    const int page = page_of(p.c, p.b, seq, t, p.status);
    if (page < 0) return;
    const unsigned parts = p.c.dim >> 4, per = parts * p.c.heads;
    const long long head_codes = static_cast<long long>(p.c.dim) << p.c.page_shift;
    const long long codes0 = code_at(p.c, page, 0, t), scale0 = scale_at(p.c, page, 0, t);
    const int head_scales = 1 << (p.c.page_shift - p.c.block_shift);
    for (unsigned x = lane; x < 2 * per; x += 128) {
        uint4 u[4];
        float s[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const unsigned y = x + 32 * i, z = y >= per ? y - per : y, head = z / parts, part = z - head * parts;
            if (y >= 2 * per) continue;
            u[i] = __ldg(reinterpret_cast<const uint4 *>((y >= per ? p.c.v : p.c.k) + codes0 + head * head_codes + 16 * part));
            s[i] = __ldg((y >= per ? p.c.vs : p.c.ks) + scale0 + head * head_scales);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const unsigned y = x + 32 * i, z = y >= per ? y - per : y, head = z / parts, part = z - head * parts;
            if (y >= 2 * per) continue;
            float v[8], w[8];
            decode4(p.c.fp8, u[i].x, v);
            decode4(p.c.fp8, u[i].y, v + 4);
            decode4(p.c.fp8, u[i].z, w);
            decode4(p.c.fp8, u[i].w, w + 4);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                v[j] *= s[i];
                w[j] *= s[i];
            }
            const Rows &o = y >= per ? p.vo : p.ko;
            const long long at = tok * o.ts + head * o.hs + 16 * part;
            store8(o, at, v);
            store8(o, at + 8, w);
        }
    }
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
    const int tile = lpt == 2 ? tile_tokens<2>() : tile_tokens<8>();
    const int block = 1 << p.c.block_shift, units = kWarps / (block / tile);
    const bool step = p.b.max_new == 1;
    const long long slots = (long long)(p.b.n_tokens / block) + 2LL * p.b.n_seqs;
    const int per_slot = (2 * p.c.heads + units - 1) / units;
    const long long step_units = 2LL * p.b.n_seqs * p.c.heads, per_cta = kWarps * (32 / lpt);
    const long long kv_ctas = step ? (step_units + per_cta - 1) / per_cta : slots * per_slot;
    const int heads_per_warp = 32 / lpt * kQPasses, parts = p.q.p ? (p.q.heads + heads_per_warp - 1) / heads_per_warp : 0;
    const long long q_units = (long long)p.b.n_tokens * parts, q_ctas = (q_units + kWarps - 1) / kWarps;
    if (kv_ctas + q_ctas >= 0x7fffffffLL || q_units > 0x7fffffffLL || step_units > 0x7fffffffLL) return cudaErrorInvalidValue;
    const unsigned grid = (unsigned)(kv_ctas + q_ctas) + !step;  // several new tokens: one CTA looks at all sequences
    if (step) {
        if (lpt == 2) k_kv_append_step<2><<<grid, kThreads, 0, s>>>(p, (int)kv_ctas, parts);
        else if (lpt == 4) k_kv_append_step<4><<<grid, kThreads, 0, s>>>(p, (int)kv_ctas, parts);
        else k_kv_append_step<8><<<grid, kThreads, 0, s>>>(p, (int)kv_ctas, parts);
        return cudaGetLastError();
    }
    if (lpt == 2) k_kv_append<2><<<grid, kThreads, 0, s>>>(p, (int)kv_ctas, per_slot, parts);
    else if (lpt == 4) k_kv_append<4><<<grid, kThreads, 0, s>>>(p, (int)kv_ctas, per_slot, parts);
    else k_kv_append<8><<<grid, kThreads, 0, s>>>(p, (int)kv_ctas, per_slot, parts);
    return cudaGetLastError();
}

cudaError_t read_back(const ReadParams &p, cudaStream_t s) {
    k_kv_read<<<(unsigned)((p.b.n_tokens + 7) / 8), 256, 0, s>>>(p);
    return cudaGetLastError();
}

}  // namespace kv
}  // namespace ditch
