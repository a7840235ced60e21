// Attention over the paged 8-bit cache for few rows per key / value head:
// single tokens, a few tokens at once, and f32 rows.
//
// The cache is read once per row tile and is all that counts (2 bytes per
// key and dimension against 4 flops per query head): the kernel has to keep
// HBM busy while it turns codes into f16, which holds every int8 and E4M3
// code exactly, and multiplies on the tensor cores (mma.sync m16n8k16; a
// tcgen05 tile would be 128 rows, of which a single token's group fills 4 to
// 8). Products are transposed, so that 8 query rows are the narrow side:
//   S^T [16 tokens][8 rows] = K codes . Q^T      (per 16-token block)
//   O^T [dims][8 rows]     += sv (V codes^T . P^T)
// with the block's scales applied to the f32 products: s = sk c_r S^T where
// c_r holds the softmax scale and the power of two by which row r of Q was
// brought into f16's range, and sv as the block's P . V is added to the f32
// sums. Codes go from global memory to registers in 16-byte pieces and from
// there to MMA operands without shared memory: the order of the reduction is
// free, so a lane's 32 (of K) or 16 (of V) contiguous dimensions are the
// ones its fragments name.
//
// Online softmax per warp in base 2. The reference maximum moves only when a
// score passes it by kLazy: weights stay below 2^kLazy, well inside f16, and
// most blocks skip the reduction over the lanes and the rescale.
//
// f32 rows: Q and P are each split into two f16 (22 bits), two MMAs for one.
//
// A sequence's blocks are split over CTAs when there are few rows; partial
// sums (f32) go to the workspace and the CTA that arrives last adds them in
// order, so results do not depend on timing.
#include <algorithm>

#include "kv_range.cuh"

namespace ditch {
namespace kv {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kBlk = 16;         // tokens of one step of a warp
constexpr float kLazy = 8.0f;
constexpr int kCounters = 16384;  // split work items: their arrival counters, first in the workspace
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ float2 half2_floats(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2 *>(&u)); }

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct Plan {
    int nt;             // tiles of 8 rows per CTA
    int row_tiles;      // CTAs over the rows of a (sequence, kv head)
    int splits, len;    // CTAs over its blocks at most, and the blocks of one
    long long items;
};

template <int DP, int NT, bool SPLIT, bool FP8>
struct Step {
    static constexpr int kK = DP / 64;  // 16-byte pieces of a key per lane
    uint4 k[2][kK];                     // tokens g and g + 8, dimensions (DP / 4) t ...
    uint32_t v[4][DP / 32];             // tokens 2t, 2t + 1, 2t + 8, 2t + 9, dimensions (DP / 8) g ...
    float sk, sv;
    int tok;                            // first token, or -1: nothing to see
};

// The codes and scales of block `blk` of the range (a page of 16 tokens or
// more holds whole blocks).
template <int DP, int NT, bool SPLIT, bool FP8>
__device__ __forceinline__ void load_step(Step<DP, NT, SPLIT, FP8> &s, const Cache &c, int head, int tok, int page, int lane) {
    using St = Step<DP, NT, SPLIT, FP8>;
    s.tok = page < 0 ? -1 : tok;
    if (page < 0) return;
    const int g = lane >> 2, t = lane & 3;
    const long long at = code_at(c, page, head, tok), sa = scale_at(c, page, head, tok);
    const uint8_t *kp = c.k + at + (long long)g * c.dim + t * (DP / 4);
    const uint8_t *vp = c.v + at + (long long)(2 * t) * c.dim + g * (DP / 8);
#pragma unroll
    for (int r = 0; r < 2; r++)
#pragma unroll
        for (int i = 0; i < St::kK; i++) {
            const bool in = t * (DP / 4) + 16 * i < c.dim;
            s.k[r][i] = in ? __ldcs(reinterpret_cast<const uint4 *>(kp + (long long)(8 * r) * c.dim + 16 * i)) : make_uint4(0, 0, 0, 0);
        }
    const bool in = g * (DP / 8) < c.dim;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const uint8_t *row = vp + (long long)((r & 1) + 8 * (r >> 1)) * c.dim;
        if (DP == 128) {
            const uint4 u = in ? __ldcs(reinterpret_cast<const uint4 *>(row)) : make_uint4(0, 0, 0, 0);
            s.v[r][0] = u.x, s.v[r][1] = u.y, s.v[r][DP / 32 - 2] = u.z, s.v[r][DP / 32 - 1] = u.w;
        } else {
            const uint2 u = in ? __ldcs(reinterpret_cast<const uint2 *>(row)) : make_uint2(0, 0);
            s.v[r][0] = u.x, s.v[r][1] = u.y;
        }
    }
    s.sk = __ldg(c.ks + sa);
    s.sv = __ldg(c.vs + sa);
}

struct Smem {
    float m[kWarps][32], l[kWarps][32];
    int last;
};

template <int DP, int NT, bool SPLIT, bool FP8>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 3 : 2) k_attend(AttendParams p, Plan plan) {
    constexpr int kRows = 8 * NT;
    constexpr int kQs = DP + 8;        // row stride of Q in shared memory (f16)
    constexpr int kSteps = DP / 16;    // MMA steps over the dimensions
    constexpr int kMt = DP / 16;       // tiles of 16 dimensions of O^T
    constexpr float kUnit = FP8 ? 256.0f : 1.0f;  // value of a code in f16
    __shared__ Smem sm;
    __shared__ __align__(16) __half s_q[(SPLIT ? 2 : 1) * kRows * kQs];
    __shared__ __align__(16) float s_o[kRows * DP];
    __shared__ float s_c[kRows];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x;
    int item = blockIdx.y + gridDim.y * blockIdx.z;  // (sequence, kv head, row tile)
    if (item >= plan.items) return;
    const int tile = item % plan.row_tiles, head = item / plan.row_tiles % p.c.heads, seq = item / plan.row_tiles / p.c.heads;
    const Span a = span_of(p.b, p.c.page_shift, seq, p.status);
    const int group = p.q.heads / p.c.heads, rows = a.n * group, r0 = tile * kRows;
    if (r0 >= rows) return;
    const int n_rows = min(kRows, rows - r0), first = a.len - a.n;
    const int p_lo = first + r0 / group, p_hi = first + (r0 + n_rows - 1) / group;
    const Range range = range_of(p_lo, p_hi, p.window, p.sinks, kBlk);
    const int per = max(plan.len, (range.n + plan.splits - 1) / plan.splits);
    const int my_splits = (range.n + per - 1) / per;
    if (split >= my_splits) return;
    const int b_lo = split * per, b_hi = min(range.n, b_lo + per);

    // this warp's blocks are b_lo + warp, + kWarps, ...; lane i looks up the page of the i-th
    int b = b_lo + warp, ahead = 0;
    int pages = -1;
    auto look_up = [&]() {
        const int x = b_lo + warp + kWarps * (ahead + lane);
        pages = x < b_hi ? page_of(p.c, p.b, seq, range.token(x, kBlk), p.status) : -1;
    };
    look_up();

    // ---- Q to f16, each row by a power of two to below 2 ----
    for (int r = warp; r < kRows; r += kWarps) {
        float x[DP / 32];
        uint32_t top = 0;
        const int row = r0 + r, i = row / group;
        const long long at = (a.row0 + i) * p.q.ts + (head * group + row - i * group) * p.q.hs;
#pragma unroll
        for (int e = 0; e < DP / 32; e++) {
            const int d = lane + 32 * e;
            x[e] = r < n_rows && d < p.c.dim ? load1(p.q, at + d) : 0.0f;
            top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        int e2 = static_cast<int>(top >> 23) - 127;
        e2 = top >= 0x7f800000u || top == 0 ? 0 : max(-120, min(120, e2));
        const float down = __uint_as_float(static_cast<uint32_t>(127 - e2) << 23);
        if (lane == 0) s_c[r] = p.scale * kLog2e * __uint_as_float(static_cast<uint32_t>(127 + e2) << 23) * kUnit;
#pragma unroll
        for (int e = 0; e < DP / 32; e++) {
            // pairs of codes are taken as (0, 2) and (1, 3) of four
            int d = lane + 32 * e;
            d = FP8 && ((d & 3) == 1 || (d & 3) == 2) ? d ^ 3 : d;
            const float y = x[e] * down;
            const __half h = __float2half_rn(y);
            s_q[r * kQs + d] = h;
            if (SPLIT) s_q[(kRows + r) * kQs + d] = __float2half_rn(y - __half2float(h));
        }
    }
    __syncthreads();

    float c_row[NT][2];
    int top_key[NT][2], low_key[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = 8 * n + 2 * t + e;
            c_row[n][e] = s_c[r];
            top_key[n][e] = r < n_rows ? first + (r0 + r) / group : -1;
            low_key[n][e] = p.window ? top_key[n][e] - p.window + 1 : 0;
        }
    uint32_t qf[NT == 1 && !SPLIT ? kSteps : 1][2];
    if (NT == 1 && !SPLIT) {
#pragma unroll
        for (int s = 0; s < kSteps; s++) {
            const uint2 u = *reinterpret_cast<const uint2 *>(s_q + g * kQs + t * (DP / 4) + 4 * s);
            qf[NT == 1 && !SPLIT ? s : 0][0] = u.x;
            qf[NT == 1 && !SPLIT ? s : 0][1] = u.y;
        }
    }

    float o[NT][kMt][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int j = 0; j < kMt; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[n][j][e] = 0.0f;
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.0f;
    }

    // The page lookups and loads of a step come one step ahead of its use.
    auto fetch = [&](Step<DP, NT, SPLIT, FP8> &s, int i) {
        const int x = b_lo + warp + kWarps * i;
        if (i - ahead >= 32) {
            ahead += 32;
            look_up();
        }
        const int page = __shfl_sync(0xffffffffu, pages, i - ahead);
        if (x < b_hi) load_step<DP, NT, SPLIT, FP8>(s, p.c, head, range.token(x, kBlk), page, lane);
        else s.tok = -1;
    };

    auto use = [&](const Step<DP, NT, SPLIT, FP8> &s) {
        if (s.tok < 0) return;
        // ---- S^T = K . Q^T ----
        float sc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) sc[n][e] = 0.0f;
#pragma unroll
        for (int i = 0; i < Step<DP, NT, SPLIT, FP8>::kK; i++) {
            const uint32_t w0[4] = {s.k[0][i].x, s.k[0][i].y, s.k[0][i].z, s.k[0][i].w};
            const uint32_t w1[4] = {s.k[1][i].x, s.k[1][i].y, s.k[1][i].z, s.k[1][i].w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t f[4];
                key_pairs<FP8>(w0[j], f[0], f[2]);
                key_pairs<FP8>(w1[j], f[1], f[3]);
                const int step = 4 * i + j;
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    if (NT == 1 && !SPLIT) {
                        mma_f16(sc[n], f, qf[NT == 1 && !SPLIT ? step : 0][0], qf[NT == 1 && !SPLIT ? step : 0][1]);
                    } else {
                        const __half *at = s_q + (8 * n + g) * kQs + t * (DP / 4) + 4 * step;
                        const uint2 u = *reinterpret_cast<const uint2 *>(at);
                        mma_f16(sc[n], f, u.x, u.y);
                        if (SPLIT) {
                            const uint2 w = *reinterpret_cast<const uint2 *>(at + kRows * kQs);
                            mma_f16(sc[n], f, w.x, w.y);
                        }
                    }
                }
            }
        }
        // ---- softmax ----
        const bool whole = s.tok + kBlk - 1 <= p_lo && (!p.window || s.tok > p_hi - p.window);
        bool sees[NT][2];
        bool over = false;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float f = s.sk * c_row[n][e];
                sc[n][e] *= f;
                sc[n][e + 2] *= f;
                sees[n][e] = true;
                if (!whole) {
                    const int hi = top_key[n][e], lo = low_key[n][e];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int key = s.tok + g + 8 * h;
                        if (key > hi || (key < lo && key >= p.sinks)) sc[n][e + 2 * h] = -INFINITY;
                    }
                    sees[n][e] = s.tok <= hi && (s.tok + kBlk > lo || s.tok < p.sinks);
                }
                over |= fmaxf(sc[n][e], sc[n][e + 2]) > m[n][e] + kLazy;
            }
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float x = fmaxf(sc[n][e], sc[n][e + 2]);
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
                    x = fmaxf(x, m[n][e]);
                    const float keep = m[n][e] == -INFINITY ? 0.0f : exp2f(m[n][e] - x);
                    m[n][e] = x;
                    l[n][e] *= keep;
#pragma unroll
                    for (int j = 0; j < kMt; j++) {
                        o[n][j][e] *= keep;
                        o[n][j][e + 2] *= keep;
                    }
                }
        }
        uint32_t pb[NT][2], pl[SPLIT ? NT : 1][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float ref = m[n][e] == -INFINITY ? 0.0f : m[n][e];
                sc[n][e] = SPLIT ? exp2f(sc[n][e] - ref) : exp2_fast(sc[n][e] - ref);
                sc[n][e + 2] = SPLIT ? exp2f(sc[n][e + 2] - ref) : exp2_fast(sc[n][e + 2] - ref);
                l[n][e] += sc[n][e] + sc[n][e + 2];
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t u = half2_bits(sc[n][2 * h], sc[n][2 * h + 1]);
                pb[n][h] = transpose8x8(u);
                if (SPLIT) {
                    const float2 f = half2_floats(u);
                    pl[SPLIT ? n : 0][h] = transpose8x8(half2_bits(sc[n][2 * h] - f.x, sc[n][2 * h + 1] - f.y));
                }
            }
        }
        // ---- O^T += sv V^T . P^T ----
        float w[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) w[n][e] = sees[n][e] ? s.sv * kUnit : 0.0f;
#pragma unroll
        for (int i = 0; i < DP / 32; i++) {
#pragma unroll
            for (int half = 0; half < 2; half++) {  // dimensions (DP / 8) g + 4 i + 2 half, + 1
                uint32_t f[4];
                value_pairs<FP8>(s.v[0][i], s.v[1][i], half, f[0], f[1]);
                value_pairs<FP8>(s.v[2][i], s.v[3][i], half, f[2], f[3]);
                const int j = 2 * i + half;
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    mma_f16(x, f, pb[n][0], pb[n][1]);
                    if (SPLIT) mma_f16(x, f, pl[SPLIT ? n : 0][0], pl[SPLIT ? n : 0][1]);
#pragma unroll
                    for (int e = 0; e < 4; e++) o[n][j][e] = fmaf(x[e], w[n][e & 1], o[n][j][e]);
                }
            }
        }
    };

    Step<DP, NT, SPLIT, FP8> s0, s1;
    const int n_steps = b < b_hi ? (b_hi - b + kWarps - 1) / kWarps : 0;
    fetch(s0, 0);
    for (int i = 0; i < n_steps; i += 2) {
        fetch(s1, i + 1);
        use(s0);
        fetch(s0, i + 2);
        use(s1);
    }

    // ---- the warps' sums, in order ----
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], x);
            if (m[n][e] == -INFINITY && l[n][e] != 0.0f) m[n][e] = INFINITY;  // only NaN scores: the row is NaN
            if (g == 0) {
                sm.m[warp][8 * n + 2 * t + e] = m[n][e];
                sm.l[warp][8 * n + 2 * t + e] = l[n][e];
            }
        }
    __syncthreads();
    float keep[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = 8 * n + 2 * t + e;
            float x = sm.m[0][r];
#pragma unroll
            for (int w = 1; w < kWarps; w++) x = fmaxf(x, sm.m[w][r]);
            keep[n][e] = m[n][e] == -INFINITY ? 0.0f : exp2f(m[n][e] - x);
        }
    for (int w = 0; w < kWarps; w++) {
        if (w == warp) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < kMt; j++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float2 *d = reinterpret_cast<float2 *>(s_o + (8 * n + 2 * t + e) * DP + g * (DP / 8) + 2 * j);
                        const float k = keep[n][e];
                        float2 v = make_float2(o[n][j][e] * k, o[n][j][e + 2] * k);
                        if (k == 0.0f) v = make_float2(0.0f, 0.0f);
                        if (w) {
                            const float2 u = *d;
                            v.x += u.x;
                            v.y += u.y;
                        }
                        *d = v;
                    }
        }
        __syncthreads();
    }

    auto row_ml = [&](int r, float &mx, float &sum) {
        mx = sm.m[0][r];
#pragma unroll
        for (int w = 1; w < kWarps; w++) mx = fmaxf(mx, sm.m[w][r]);
        sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; w++) sum += sm.m[w][r] == -INFINITY ? 0.0f : sm.l[w][r] * exp2f(sm.m[w][r] - mx);
    };
    auto put = [&](int r, int d, float v) {
        const int row = r0 + r, i = row / group;
        store1(p.out, (a.row0 + i) * p.out.ts + (head * group + row - i * group) * p.out.hs + d, v);
    };
    if (my_splits == 1) {
        for (int x = tid; x < n_rows * DP; x += kThreads) {
            const int r = x / DP, d = x - r * DP;
            if (d >= p.c.dim) continue;
            float mx, sum;
            row_ml(r, mx, sum);
            put(r, d, mx == -INFINITY ? 0.0f : s_o[r * DP + d] / sum);
        }
        return;
    }
    // partial sums of this split: rows of DP sums, then maxima and sums
    float *ws = reinterpret_cast<float *>(static_cast<uint8_t *>(p.ws) + kCounters * sizeof(int));
    constexpr int kPart = kRows * (DP + 2);
    float *part = ws + (static_cast<long long>(item) * plan.splits + split) * kPart;
    for (int x = tid; x < kRows * DP; x += kThreads) part[x] = s_o[x];
    if (tid < kRows) {
        float mx, sum;
        row_ml(tid, mx, sum);
        part[kRows * DP + tid] = mx;
        part[kRows * DP + kRows + tid] = sum;
    }
    __threadfence();
    __syncthreads();
    if (tid == 0) {
        int *count = static_cast<int *>(p.ws) + item;
        sm.last = atomicAdd(count, 1) == my_splits - 1;
        if (sm.last) *count = 0;
    }
    __syncthreads();
    if (!sm.last) return;
    __threadfence();
    const float *all = ws + static_cast<long long>(item) * plan.splits * kPart;
    for (int x = tid; x < n_rows * DP; x += kThreads) {
        const int r = x / DP, d = x - r * DP;
        float mx = -INFINITY;
        for (int s = 0; s < my_splits; s++) mx = fmaxf(mx, __ldcg(all + s * kPart + kRows * DP + r));
        float sum = 0.0f, v = 0.0f;
        for (int s = 0; s < my_splits; s++) {
            const float ms = __ldcg(all + s * kPart + kRows * DP + r);
            if (ms == -INFINITY) continue;
            const float k = exp2f(ms - mx);
            sum = fmaf(k, __ldcg(all + s * kPart + kRows * DP + kRows + r), sum);
            v = fmaf(k, __ldcg(all + s * kPart + x), v);
        }
        if (d < p.c.dim) put(r, d, mx == -INFINITY ? 0.0f : v / sum);
    }
}

// CTAs of 4 warps, three to an SM (two for more than 8 rows). A sequence is
// split until there are about kWaves rounds of CTAs, so that ragged lengths
// leave no SM idle for long, but not below kMinTokens once every SM has
// work, and not below one block per warp before that.
constexpr int kWaves = 12, kMinTokens = 512;

Plan plan_of(const Cache &c, const Batch &b, int q_heads, int sms, bool split_f32, int seen) {
    Plan p;
    const long long rows = (long long)b.max_new * (q_heads / c.heads);
    p.nt = rows <= 8 ? 1 : rows <= 16 || split_f32 ? 2 : 4;
    p.row_tiles = (int)((rows + 8 * p.nt - 1) / (8 * p.nt));
    p.items = (long long)b.n_seqs * c.heads * p.row_tiles;
    const int tokens = seen;
    const long long want = ((long long)sms * 3 * kWaves + p.items - 1) / p.items;
    long long len = std::max<long long>((tokens + want - 1) / want, kBlk * kWarps);
    if (p.items >= sms) len = std::max<long long>(len, kMinTokens);
    p.len = (int)((len + kBlk - 1) / kBlk);
    p.splits = p.items > kCounters ? 1 : (tokens + p.len * kBlk - 1) / (p.len * kBlk);
    return p;
}

template <int DP, int NT, bool SPLIT>
cudaError_t launch2(const AttendParams &p, const Plan &plan, cudaStream_t s) {
    const long long ny = std::min<long long>(plan.items, 32768), nz = (plan.items + ny - 1) / ny;
    if (nz > 65535) return cudaErrorInvalidValue;
    const dim3 grid(plan.splits, (unsigned)ny, (unsigned)nz);
    if (p.c.fp8) k_attend<DP, NT, SPLIT, true><<<grid, kThreads, 0, s>>>(p, plan);
    else k_attend<DP, NT, SPLIT, false><<<grid, kThreads, 0, s>>>(p, plan);
    return cudaGetLastError();
}

template <int DP>
cudaError_t launch1(const AttendParams &p, const Plan &plan, bool split_f32, cudaStream_t s) {
    if (split_f32) return plan.nt == 1 ? launch2<DP, 1, true>(p, plan, s) : launch2<DP, 2, true>(p, plan, s);
    return plan.nt == 1 ? launch2<DP, 1, false>(p, plan, s) : plan.nt == 2 ? launch2<DP, 2, false>(p, plan, s) : launch2<DP, 4, false>(p, plan, s);
}

size_t plan_bytes(const Cache &c, const Plan &p) {
    if (p.splits <= 1) return 0;
    const size_t dp = c.dim <= 64 ? 64 : 128;
    return kCounters * sizeof(int) + (size_t)p.items * p.splits * (8 * p.nt) * (dp + 2) * sizeof(float);
}

}  // namespace

size_t attend_workspace(const Cache &c, const Batch &b, int q_heads, int sms) {
    return std::max(plan_bytes(c, plan_of(c, b, q_heads, sms, false, b.max_len)),
                    plan_bytes(c, plan_of(c, b, q_heads, sms, true, b.max_len)));
}

cudaError_t attend(const AttendParams &p, int sms, cudaStream_t s) {
    const bool split_f32 = p.out.dtype == kF32;
    // keys that a row tile can see, at most; no more than the workspace was sized for
    long long seen = p.b.max_len;
    if (p.window) seen = std::min<long long>(seen, (long long)p.window + p.sinks + p.b.max_new);
    const Plan plan = plan_of(p.c, p.b, p.q.heads, sms, split_f32, (int)seen);
    return p.c.dim <= 64 ? launch1<64>(p, plan, split_f32, s) : launch1<128>(p, plan, split_f32, s);
}

}  // namespace kv
}  // namespace ditch
