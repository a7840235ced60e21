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
// sums. int8 keys are not converted at all: Q is taken as a 23-bit fixed-point
// number of three signed 8-bit digits and multiplied with m16n8k32 integer
// MMAs, exactly (three MMAs for what would be two in f16, but no work per
// code). Each warp keeps a ring of pairs of blocks of its own in shared
// memory, filled by TMA one pair ahead (a box of 16 tokens, rows padded with
// zeros to 64 or 128 bytes, swizzled so that the reads below meet no bank
// twice), and waits for nobody else. Two blocks at a time give the chains of
// dependent MMAs company. The order of the reduction is free, so a lane's 32
// (of K) or 16 (of V) contiguous dimensions are the ones its fragments name.
//
// Online softmax per warp in base 2. The reference maximum moves only when a
// score passes it by lazy(): most blocks skip the reduction over the lanes and
// the rescale. Weights are taken times 2^(15 - lazy()), which fills f16 up to
// 2^15 and leaves f16's normal numbers, and with them the weights' precision,
// down to 2^-21 (16 bits out) or 2^-27 of the reference: beside a sink that has
// nearly all weight, and hardly a value, the others are as small. f32 rows are
// the more exact the less is left for the lazy maximum (two halves resolve
// 2^-24 of f16's unit, whichever they are of).
//
// Measured: one row for each of 32 sequences of 4000 to 32000 tokens (1.01 GB
// of E4M3 codes and scales) in 169 to 177 us on five boxes, 5.7 to 6.0 TB/s,
// 0.87 to 0.91 of the copy bandwidth; 64 sequences with 1028 tokens in sight
// (135 MB, int8) in 42 us, 3.2 TB/s, where the beginning and end of each item
// show. With codes loaded straight
// into registers instead of by TMA the first took 330 us.
//
// f32 out: P (and Q over an E4M3 cache) is split into two f16 (22 bits), two
// MMAs for one. 16 bits out take both as one f16, f32 queries over an E4M3
// cache as well: the split costs those 7 to 30 % (32 sequences of 16000 tokens
// 175 us, with it 189; 128 of 1500 tokens on one head 17 and 22 us).
//
// The blocks of all work items (sequence, key / value head, row tile), one
// item after another, are divided evenly over as many CTAs as the GPU holds,
// whatever the sequences' lengths. A CTA's share may begin and end inside an
// item: it leaves that item's sums (f32) in the workspace, and the CTA that
// brings an item's last part adds the parts in order, so results do not
// depend on timing. Short items are taken whole instead, one by each CTA,
// where that is done sooner (ITEMS): no parts, no counting of sequences.
#include <algorithm>

#include "gemm.cuh"
#include "kv_range.cuh"

namespace ditch {
namespace kv {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kBlk = 16;         // tokens of a block: what one MMA takes
constexpr int kMinBlocks = 8;    // of a CTA's share: a pair for each warp
constexpr float kTop = 15.0f;    // weights in P are below 2^kTop
constexpr int kCounters = 4096;  // arrival counters (one per CTA), first in the workspace
constexpr float kLog2e = 1.4426950408889634f;

constexpr float lazy(bool split) { return split ? 2.0f : 8.0f; }

// d = a b + c
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
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

// A warp's ring: kDepth pairs of blocks of K and V codes, rows of DP bytes swizzled by
// TMA (16-byte chunk c of row r lies at c ^ (r & 7) for 128-byte rows, at
// c ^ (r / 2 & 3) for 64-byte rows).
constexpr int kDepth = 2;

template <int DP>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
    return r * DP + ((DP == 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) << 4);
}

__device__ __forceinline__ void tma_load_3d(const CUtensorMap *map, uint64_t *bar, void *dst, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(y), "r"(z)
        : "memory");
}

// Two f32 in a 64-bit register, for the packed arithmetic.
using f32x2 = unsigned long long;

__device__ __forceinline__ f32x2 pack(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float2 unpack(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}

__device__ __forceinline__ void fma2(f32x2 &d, f32x2 a, f32x2 b) { asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(d) : "l"(a), "l"(b)); }

__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ uint4 lds128(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}

__device__ __forceinline__ uint2 lds64(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
    return v;
}

struct Smem {
    uint64_t full[kWarps][kDepth];
    float m[kWarps][32], l[kWarps][32], k[kWarps][32];
    long long sums[kWarps], at;
    int seq, last, abort;
};

// CTAs of four warps to an SM, by their registers.
template <int NT, bool SPLIT>
constexpr int ctas_per_sm() {
    return NT == 1 ? 3 : 2;
}

// Shared memory from a 1024-byte aligned base: the rings, over which the
// warps' sums go at the end of an item, and Q.
template <int DP, int NT, bool SPLIT>
struct Layout {
    static constexpr int kTile = kBlk * DP;  // bytes of a block's K or V
    static constexpr int kStage = 4 * kTile;  // K, V of the first block, K, V of the second
    static constexpr int kRing = kWarps * kDepth * kStage;
    static constexpr int kO = kWarps * 8 * NT * DP * 4;
    static constexpr int kQf16 = (SPLIT ? 2 : 1) * 8 * NT * (DP + 8) * 2, kQdigits = 3 * 8 * NT * (DP + 16);
    static constexpr int kQ = ((kQf16 > kQdigits ? kQf16 : kQdigits) + 15) & ~15;
    static constexpr int kQAt = kRing > kO ? kRing : kO;
    static constexpr int kBytes = 1024 + kQAt + kQ;
};

// A sequence's work: row tiles per head, and block slots of each (an upper
// bound where there are several tiles; slots past a tile's blocks are empty).
struct Work {
    Span a;
    int tiles, slots;
};

template <int ROWS>
__device__ __forceinline__ Work work_of(const AttendParams &p, int group, int seq) {
    Work w;
    w.a = span_of(p.b, p.c.page_shift, seq, p.status);
    w.tiles = (w.a.n * group + ROWS - 1) / ROWS;
    w.slots = 0;
    if (w.tiles == 1) {
        w.slots = range_of(w.a.len - w.a.n, w.a.len - 1, p.window, p.sinks, kBlk).n;
    } else if (w.tiles > 1) {
        const long long all = (w.a.len - 1) / kBlk + 1;
        const long long some = (p.sinks + kBlk - 1) / kBlk + (static_cast<long long>(p.window) + ROWS / group + 1) / kBlk + 2;
        w.slots = static_cast<int>(p.window && some < all ? some : all);
    }
    return w;
}

template <int DP, int NT, bool SPLIT, bool FP8, bool ITEMS>
__global__ void __launch_bounds__(kThreads, ctas_per_sm<NT, SPLIT>())
    k_attend(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, AttendParams p) {
    using L = Layout<DP, NT, SPLIT>;
    constexpr int kRows = 8 * NT;
    constexpr int kQs = DP + 8;        // row stride of Q in shared memory (f16)
    constexpr int kQd = DP + 16;       // row stride of Q's digits (bytes)
    constexpr int kSteps = FP8 ? DP / 16 : DP / 32;  // MMA steps over the dimensions
    constexpr bool kQRegs = NT == 1 && (!SPLIT || !FP8);  // Q's fragments stay in registers
    constexpr int kDigits = FP8 ? 1 : 3;
    constexpr int kMt = DP / 16;       // tiles of 16 dimensions of O^T
    constexpr float kLazy = lazy(SPLIT);
    constexpr int kPart = kRows * (DP + 2);   // floats of a part: sums, maxima, sums of weights
    extern __shared__ uint8_t smem_raw[];
    __shared__ Smem sm;
    __shared__ float s_c[kRows];
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    __half *s_q = reinterpret_cast<__half *>(base + L::kQAt);
    const int group = p.q.heads / p.c.heads;
    int8_t *s_d = reinterpret_cast<int8_t *>(s_q);
    uint8_t *ring = base + warp * (kDepth * L::kStage);
    // where this lane's pieces lie in a K and in a V tile (+ 8 rows: + 8 DP)
    uint32_t k_at[DP / 64], v_at[2];
#pragma unroll
    for (int i = 0; i < DP / 64; i++) k_at[i] = chunk_at<DP>(g, t * (DP / 64) + i);
#pragma unroll
    for (int r = 0; r < 2; r++) v_at[r] = chunk_at<DP>(2 * t + r, DP == 128 ? g : g >> 1) + (DP == 128 ? 0 : 8 * (g & 1));
    uint64_t *full = sm.full[warp];
    if (lane == 0) {
        for (int i = 0; i < kDepth; i++) mbar_init(&full[i], 1);
        fence_barrier_init();
    }
    if (tid == 0) sm.abort = 0;

    int seq = 0, item = 0, off = 0;
    Work work;
    long long pos = 0, end = 1, per = 1;
    if constexpr (!ITEMS) {
        // ---- this CTA's share of the block slots: [pos, end) ----
        const int chunk = (p.b.n_seqs + kThreads - 1) / kThreads;  // sequences a thread counts
        const int c_lo = min(tid * chunk, p.b.n_seqs), c_hi = min(c_lo + chunk, p.b.n_seqs);
        long long mine = 0;
        for (int x = c_lo; x < c_hi; x++) {
            const Work w = work_of<kRows>(p, group, x);
            mine += static_cast<long long>(w.tiles) * w.slots * p.c.heads;
        }
        long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        if (lane == 31) sm.sums[warp] = upto;
        __syncthreads();
        long long total = 0;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            if (w < warp) upto += sm.sums[w];
            total += sm.sums[w];
        }
        per = max((total + gridDim.x - 1) / gridDim.x, static_cast<long long>(kMinBlocks));
        pos = per * blockIdx.x;
        end = min(total, pos + per);
        if (pos >= end) return;
        if (upto - mine <= pos && pos < upto) {
            long long at = upto - mine;
            int x = c_lo;
            for (;; x++) {
                const Work w = work_of<kRows>(p, group, x);
                const long long n = static_cast<long long>(w.tiles) * w.slots * p.c.heads;
                if (pos < at + n) break;
                at += n;
            }
            sm.seq = x;
            sm.at = at;
        }
        __syncthreads();
        seq = sm.seq;
        work = work_of<kRows>(p, group, seq);
        item = static_cast<int>((pos - sm.at) / work.slots);  // of the sequence: head * tiles + tile
        off = static_cast<int>(pos - sm.at - static_cast<long long>(item) * work.slots);
    } else {
        // items are (sequence, head), dealt out to the CTAs
        __syncthreads();
        pos = blockIdx.x;
        end = static_cast<long long>(p.b.n_seqs) * p.c.heads;
    }

    const int page_mask = (1 << p.c.page_shift) - 1;
    uint32_t phase = 0;  // bit st: parity of the next completion of stage st
    int st = 0;          // the ring's next stage
    bool dead = false;   // a wait ran out

    while (pos < end) {
        if constexpr (ITEMS) {
            seq = static_cast<int>(pos / p.c.heads);
            item = static_cast<int>(pos - static_cast<long long>(seq) * p.c.heads);
            work = work_of<kRows>(p, group, seq);
            if (work.slots == 0) {
                pos += gridDim.x;
                continue;
            }
        }
        const Span a = work.a;
        const int n_slots = ITEMS ? work.slots : static_cast<int>(min(static_cast<long long>(work.slots - off), end - pos));
        const int head = ITEMS || work.tiles == 1 ? item : item / work.tiles, tile = item - head * work.tiles;
        const int rows = a.n * group, r0 = ITEMS ? 0 : tile * kRows, n_rows = min(kRows, rows - r0), first = a.len - a.n;
        // row r of the tile is query (skip + r) mod group of the tile's token t0 + (skip + r) / group
        const int t0 = r0 ? r0 / group : 0, skip = r0 - t0 * group;
        const float per_group = 1.0f / group;
        auto tok_of = [&](int r) { return static_cast<int>((skip + r + 0.5f) * per_group); };  // exact: skip + r < 2^17
        const int p_lo = first + t0, p_hi = p_lo + tok_of(n_rows - 1);
        const Range range = range_of(p_lo, p_hi, p.window, p.sinks, kBlk);
        const int b_lo = off, b_hi = min(range.n, off + n_slots);

        // ---- Q rows into registers ----
        // (lane l has dimensions 4 l .. 4 l + 3)
        constexpr int kMine = kRows / kWarps;
        float4 qx[kMine];
        const int d4 = 4 * lane;
#pragma unroll
        for (int i = 0; i < kMine; i++) {
            const int r = warp + kWarps * i, tok = tok_of(r);
            const long long at = (a.row0 + t0 + tok) * p.q.ts + (head * group + skip + r - tok * group) * p.q.hs;
            qx[i] = r < n_rows && d4 < p.c.dim ? load4(p.q, at + d4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        // ---- this warp's pairs of blocks: b_lo + 2 (warp + 4 i), + 1; lane 2 j + u looks up the
        // page and scales of block u of the (ahead + j)-th pair, half a window before they are used ----
        struct Look {
            int page;
            float sk, sv;
        };
        auto look_up = [&](int from) {
            Look k;
            const int x = b_lo + 2 * (warp + kWarps * (from + (lane >> 1))) + (lane & 1);
            const int tok = range.token(x, kBlk);
            k.page = x < b_hi ? page_of(p.c, p.b, seq, tok, p.status) : -1;
            k.sk = k.sv = 0.0f;
            if (k.page >= 0) {
                const long long sa = scale_at(p.c, k.page, head, tok);
                k.sk = __ldg(p.c.ks + sa);
                k.sv = __ldg(p.c.vs + sa);
            }
            return k;
        };
        int ahead = 0;
        Look look = look_up(0), later;
        later.page = -1;
        // a pair under way: first tokens (-1: nothing to see) and scales
        struct Under {
            int tok[2];
            float sk[2], sv[2];
        };
        auto start = [&](int stage, int i, Under &u) {
            if (i - ahead == 8) later = look_up(ahead + 16);
            if (i - ahead == 16) {
                ahead += 16;
                look = later;
            }
            int page[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                page[h] = __shfl_sync(0xffffffffu, look.page, 2 * (i - ahead) + h);
                u.tok[h] = page[h] < 0 ? -1 : range.token(b_lo + 2 * (warp + kWarps * i) + h, kBlk);
            }
            const int n = (page[0] >= 0) + (page[1] >= 0);
            if (n && lane == 0) {
                uint8_t *at = ring + stage * L::kStage;
                mbar_arrive_expect_tx(&full[stage], n * 2 * L::kTile);
#pragma unroll
                for (int h = 0; h < 2; h++)
                    if (page[h] >= 0) {
                        const int y = (head << p.c.page_shift) + (u.tok[h] & page_mask);
                        tma_load_3d(&k_map, &full[stage], at + 2 * h * L::kTile, y, page[h]);
                        tma_load_3d(&v_map, &full[stage], at + (2 * h + 1) * L::kTile, y, page[h]);
                    }
            }
        };
        auto scales = [&](int i, Under &u) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                u.sk[h] = __shfl_sync(0xffffffffu, look.sk, 2 * (i - ahead) + h);
                u.sv[h] = __shfl_sync(0xffffffffu, look.sv, 2 * (i - ahead) + h);
            }
        };

        Under u0, u1;
        start(st, 0, u0);
        start(st ^ 1, 1, u1);
        scales(0, u0);
        scales(1, u1);
#pragma unroll
        for (int i = 0; i < kMine; i++) {  // each row by a power of two to below 2
            const int r = warp + kWarps * i;
            const float x[4] = {qx[i].x, qx[i].y, qx[i].z, qx[i].w};
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
            top = __reduce_max_sync(0xffffffffu, top);
            int e2 = static_cast<int>(top >> 23) - 127;
            e2 = top >= 0x7f800000u || top == 0 ? 0 : max(-120, min(FP8 ? 120 : 127, e2));  // (f16 holds 2^8, the digits no more than 2)
            const float down = e2 == 127 ? 0x1p-127f : __uint_as_float(static_cast<uint32_t>(127 - e2) << 23);
            if (lane == 0) {
                float c = p.scale * kLog2e * (FP8 ? 1.0f : 0x1p-21f) * __uint_as_float(static_cast<uint32_t>(127 + e2) << 23);
                if (!FP8 && top >= 0x7f800000u) c = __uint_as_float(0x7fc00000u);
                s_c[r] = c;
            }
            if (d4 >= DP) continue;
            if (FP8) {
                const uint2 h = make_uint2(half2_bits(x[0] * down, x[1] * down), half2_bits(x[2] * down, x[3] * down));
                *reinterpret_cast<uint2 *>(s_q + r * kQs + d4) = h;
                if (SPLIT) {
                    const float2 h0 = half2_floats(h.x), h1 = half2_floats(h.y);
                    *reinterpret_cast<uint2 *>(s_q + (kRows + r) * kQs + d4) =
                        make_uint2(half2_bits(x[0] * down - h0.x, x[1] * down - h0.y), half2_bits(x[2] * down - h1.x, x[3] * down - h1.y));
                }
            } else {  // |x down| < 2: 23 bits, digits of the sum 65536 d2 + 256 d1 + d0
                uint32_t digit[3] = {0, 0, 0};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int v = __float2int_rn(x[e] * down * 0x1p21f);
                    const int d0 = static_cast<int8_t>(v), v1 = (v - d0) >> 8, d1 = static_cast<int8_t>(v1), d2 = (v1 - d1) >> 8;
                    digit[0] |= (d0 & 0xff) << (8 * e);
                    digit[1] |= (d1 & 0xff) << (8 * e);
                    digit[2] |= (d2 & 0xff) << (8 * e);
                }
#pragma unroll
                for (int d = 0; d < 3; d++) *reinterpret_cast<uint32_t *>(s_d + (d * kRows + r) * kQd + d4) = digit[d];
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
                top_key[n][e] = r < n_rows ? p_lo + tok_of(r) : -1;
                low_key[n][e] = p.window ? top_key[n][e] - p.window + 1 : 0;
            }
        auto q_frag = [&](int n, int step, int part) {  // part: low half of SPLIT's f16, or the digit
            return FP8 ? *reinterpret_cast<const uint2 *>(s_q + (part * kRows + 8 * n + g) * kQs + t * (DP / 4) + 4 * step)
                       : *reinterpret_cast<const uint2 *>(s_d + (part * kRows + 8 * n + g) * kQd + t * (DP / 4) + 8 * step);
        };
        uint2 qf[kQRegs ? kSteps : 1][kDigits];
        if (kQRegs) {
#pragma unroll
            for (int s = 0; s < kSteps; s++)
#pragma unroll
                for (int d = 0; d < kDigits; d++) qf[kQRegs ? s : 0][d] = q_frag(0, s, d);
        }

        // o[n][j]: rows 2t and 2t + 1 of dimension (DP / 8) g + 2 j, then of the next one
        f32x2 o[NT][kMt][2];
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int j = 0; j < kMt; j++)
                o[n][j][0] = o[n][j][1] = 0;
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.0f;
        }

        auto use = [&](int stage, const Under &s) {
            if ((s.tok[0] < 0 && s.tok[1] < 0) || dead) return;
            if (!mbar_wait_warp(&full[stage], (phase >> stage) & 1, &sm.abort, p.status)) {
                dead = true;
                return;
            }
            phase ^= 1u << stage;
            const uint32_t tiles = smem_u32(ring) + stage * L::kStage;
            // ---- S^T = K . Q^T ----
            float sc[2][NT][4];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const uint32_t kt = tiles + 2 * u * L::kTile;
                uint32_t w0[DP / 16], w1[DP / 16];  // tokens g and g + 8, dimensions (DP / 4) t ...
#pragma unroll
                for (int i = 0; i < DP / 64; i++) {
                    const uint4 k0 = lds128(kt + k_at[i]), k1 = lds128(kt + k_at[i] + 8 * DP);
                    w0[4 * i] = k0.x, w0[4 * i + 1] = k0.y, w0[4 * i + 2] = k0.z, w0[4 * i + 3] = k0.w;
                    w1[4 * i] = k1.x, w1[4 * i + 1] = k1.y, w1[4 * i + 2] = k1.z, w1[4 * i + 3] = k1.w;
                }
                if constexpr (FP8) {
                    // (even and odd steps apart: two chains of dependent MMAs)
                    float odd[NT][4];
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) sc[u][n][e] = odd[n][e] = 0.0f;
#pragma unroll
                    for (int i = 0; i < kSteps; i++) {
                        uint32_t f[4];
                        e4m3_pairs(w0[i], f[0], f[2]);
                        e4m3_pairs(w1[i], f[1], f[3]);
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            float(&acc)[4] = i & 1 ? odd[n] : sc[u][n];
                            const uint2 b = kQRegs ? qf[kQRegs ? i : 0][0] : q_frag(n, i, 0);
                            mma_f16(acc, f, b.x, b.y, acc);
                            if (SPLIT) {
                                const uint2 low = q_frag(n, i, 1);
                                mma_f16(acc, f, low.x, low.y, acc);
                            }
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) sc[u][n][e] += odd[n][e];
                } else {
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        int acc[3][4];
#pragma unroll
                        for (int d = 0; d < 3; d++)
#pragma unroll
                            for (int e = 0; e < 4; e++) acc[d][e] = 0;
#pragma unroll
                        for (int i = 0; i < kSteps; i++) {
                            const uint32_t f[4] = {w0[2 * i], w1[2 * i], w0[2 * i + 1], w1[2 * i + 1]};
#pragma unroll
                            for (int d = 0; d < 3; d++) {
                                const uint2 b = kQRegs ? qf[kQRegs ? i : 0][FP8 ? 0 : d] : q_frag(n, i, d);
                                mma_s8(acc[d], f, b.x, b.y);
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            sc[u][n][e] = fmaf(static_cast<float>(acc[2][e] * 256 + acc[1][e]), 256.0f, static_cast<float>(acc[0][e]));
                    }
                }
            }
            // ---- softmax ----
            bool whole[2], sees[2][NT][2];
            bool over = false;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                whole[u] = s.tok[u] >= 0 && s.tok[u] + kBlk - 1 <= p_lo && (!p.window || s.tok[u] > p_hi - p.window);
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float f = s.sk[u] * c_row[n][e];
                        sc[u][n][e] *= f;
                        sc[u][n][e + 2] *= f;
                        sees[u][n][e] = true;
                    }
                if (!whole[u]) {
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const int hi = s.tok[u] < 0 ? -2 : top_key[n][e], lo = low_key[n][e];
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                const int key = s.tok[u] + g + 8 * h;
                                if (key > hi || (key < lo && key >= p.sinks)) sc[u][n][e + 2 * h] = -INFINITY;
                            }
                            sees[u][n][e] = s.tok[u] <= hi && (s.tok[u] + kBlk > lo || s.tok[u] < p.sinks);
                        }
                }
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) over |= fmaxf(sc[u][n][e], sc[u][n][e + 2]) > m[n][e] + kLazy;
            }
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float keep[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float x = fmaxf(fmaxf(sc[0][n][e], sc[0][n][e + 2]), fmaxf(sc[1][n][e], sc[1][n][e + 2]));
#pragma unroll
                        for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
                        x = fmaxf(x, m[n][e]);
                        keep[e] = m[n][e] == -INFINITY ? 0.0f : exp2f(m[n][e] - x);
                        m[n][e] = x;
                        l[n][e] *= keep[e];
                    }
                    const f32x2 k2 = pack(keep[0], keep[1]);
#pragma unroll
                    for (int j = 0; j < kMt; j++) {
                        o[n][j][0] = mul2(o[n][j][0], k2);
                        o[n][j][1] = mul2(o[n][j][1], k2);
                    }
                }
            }
            uint32_t pb[2][NT][2], pl[2][SPLIT ? NT : 1][2];
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float ref = m[n][e] == -INFINITY ? 0.0f : m[n][e] - (kTop - kLazy);
                        sc[u][n][e] = exp2_fast(sc[u][n][e] - ref);
                        sc[u][n][e + 2] = exp2_fast(sc[u][n][e + 2] - ref);
                        l[n][e] += sc[u][n][e] + sc[u][n][e + 2];
                    }
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t b = half2_bits(sc[u][n][2 * h], sc[u][n][2 * h + 1]);
                        pb[u][n][h] = transpose8x8(b);
                        if (SPLIT) {
                            const float2 f = half2_floats(b);
                            pl[u][SPLIT ? n : 0][h] = transpose8x8(half2_bits(sc[u][n][2 * h] - f.x, sc[u][n][2 * h + 1] - f.y));
                        }
                    }
                }
            // ---- O^T += sv V^T . P^T ----
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const uint32_t vt = tiles + (2 * u + 1) * L::kTile;
                const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                f32x2 w[NT];
#pragma unroll
                for (int n = 0; n < NT; n++) w[n] = pack(sees[u][n][0] ? s.sv[u] : 0.0f, sees[u][n][1] ? s.sv[u] : 0.0f);
                // (an E4M3 NaN in memory past the sequence must not meet a weight of 0)
                const int seen = whole[u] || !FP8 ? kBlk : s.tok[u] < 0 ? 0 : p_hi + 1 - s.tok[u];
                uint32_t v[4][DP / 32];  // tokens 2t, 2t + 1, 2t + 8, 2t + 9, dimensions (DP / 8) g ...
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const uint32_t at = vt + v_at[r & 1] + (r >> 1) * 8 * DP;
                    if (DP == 128) {
                        const uint4 x = lds128(at);
                        v[r][0] = x.x, v[r][1] = x.y, v[r][DP / 32 - 2] = x.z, v[r][DP / 32 - 1] = x.w;
                    } else {
                        const uint2 x = lds64(at);
                        v[r][0] = x.x, v[r][1] = x.y;
                    }
                    if (FP8 && 2 * t + (r & 1) + 8 * (r >> 1) >= seen) {
#pragma unroll
                        for (int i = 0; i < DP / 32; i++) v[r][i] = 0;
                    }
                }
#pragma unroll
                for (int i = 0; i < DP / 32; i++) {
#pragma unroll
                    for (int half = 0; half < 2; half++) {  // dimensions (DP / 8) g + 4 i + 2 half, + 1
                        uint32_t f[4];
                        value_pairs<FP8>(v[0][i], v[1][i], half, f[0], f[1]);
                        value_pairs<FP8>(v[2][i], v[3][i], half, f[2], f[3]);
                        const int j = 2 * i + half;
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            float x[4];
                            mma_f16(x, f, pb[u][n][0], pb[u][n][1], zero);
                            if (SPLIT) mma_f16(x, f, pl[u][SPLIT ? n : 0][0], pl[u][SPLIT ? n : 0][1], x);
                            fma2(o[n][j][0], pack(x[0], x[1]), w[n]);
                            fma2(o[n][j][1], pack(x[2], x[3]), w[n]);
                        }
                    }
                }
            }
        };

        const int n_pairs = (b_hi - b_lo + 1) / 2, n_steps = warp < n_pairs ? (n_pairs - warp + kWarps - 1) / kWarps : 0;
#pragma unroll 1
        for (int i = 0; i < n_steps; i++) {
            use(st, u0);
            __syncwarp();  // every lane has read the stage
            u0 = u1;
            start(st, i + kDepth, u1);
            scales(i + kDepth, u1);
            st ^= 1;
        }
        if (dead)  // the loads under way get 0.1 ms before the memory goes to others
            for (int x = 0; x < 100; x++) __nanosleep(1000);

#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], x);
                if (m[n][e] == -INFINITY && l[n][e] != 0.0f) m[n][e] = INFINITY;  // only NaN scores: the row is NaN
            }
        // four values of row r of the tile
        auto put = [&](int r, int d, float4 v) {
            const int tok = tok_of(r);
            const long long at = (a.row0 + t0 + tok) * p.out.ts + (head * group + skip + r - tok * group) * p.out.hs + d;
            if (d >= p.c.dim) return;
            if (p.out.vec) {
                store4(p.out, at, v);
            } else {
                store1(p.out, at, v.x);
                store1(p.out, at + 1, v.y);
                store1(p.out, at + 2, v.z);
                store1(p.out, at + 3, v.w);
            }
        };
        // ---- the warps' sums, in order ----
        if (g == 0) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    sm.m[warp][8 * n + 2 * t + e] = m[n][e];
                    sm.l[warp][8 * n + 2 * t + e] = l[n][e];
                }
        }
        __syncthreads();  // the rings are no longer read: the sums go over them
        float *s_o = reinterpret_cast<float *>(base) + warp * kRows * DP;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < kMt; j += 2) {
                const float2 a0 = unpack(o[n][j][0]), a1 = unpack(o[n][j][1]), a2 = unpack(o[n][j + 1][0]), a3 = unpack(o[n][j + 1][1]);
                float4 *at = reinterpret_cast<float4 *>(s_o + (8 * n + 2 * t) * DP + g * (DP / 8) + 2 * j);
                at[0] = make_float4(a0.x, a1.x, a2.x, a3.x);
                at[DP / 4] = make_float4(a0.y, a1.y, a2.y, a3.y);
            }
        const bool alone = ITEMS || (off == 0 && n_slots == work.slots);
        const long long item_at = pos - off;
        const int c0 = static_cast<int>(item_at / per), c1 = static_cast<int>((item_at + work.slots - 1) / per);
        float *parts = reinterpret_cast<float *>(static_cast<uint8_t *>(p.ws) + kCounters * sizeof(int));
        float *part = parts + (2 * blockIdx.x + (static_cast<int>(blockIdx.x) == c0 ? 1 : 0)) * static_cast<long long>(kPart);
        if (tid < kRows) {
            float mx = sm.m[0][tid], sum = 0.0f;
#pragma unroll
            for (int w = 1; w < kWarps; w++) mx = fmaxf(mx, sm.m[w][tid]);
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float k = sm.m[w][tid] == -INFINITY ? 0.0f : exp2f(sm.m[w][tid] - mx);
                sm.k[w][tid] = k;
                sum += sm.l[w][tid] * k;
            }
            if (alone) {
                const float inv = mx == -INFINITY ? 0.0f : 1.0f / sum;
#pragma unroll
                for (int w = 0; w < kWarps; w++) sm.k[w][tid] *= inv;
            } else {
                part[kRows * DP + tid] = mx;
                part[kRows * DP + kRows + tid] = sum;
            }
        }
        __syncthreads();
        const float *all = reinterpret_cast<const float *>(base);
        for (int x = 4 * tid; x < n_rows * DP; x += 4 * kThreads) {
            const int r = x / DP;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float k = sm.k[w][r];
                const float4 u = *reinterpret_cast<const float4 *>(all + w * kRows * DP + x);
                if (k != 0.0f) {  // (a warp that saw nothing of the row)
                    v.x = fmaf(k, u.x, v.x);
                    v.y = fmaf(k, u.y, v.y);
                    v.z = fmaf(k, u.z, v.z);
                    v.w = fmaf(k, u.w, v.w);
                }
            }
            if (alone) put(r, x - r * DP, v);
            else *reinterpret_cast<float4 *>(part + x) = v;
        }
        if (!alone) {
            __syncthreads();
            if (tid == 0) {
                __threadfence();  // the CTA's part is written before it is counted
                int *count = static_cast<int *>(p.ws) + c0;
                sm.last = atomicAdd(count, 1) == c1 - c0;
                if (sm.last) *count = 0;
                __threadfence();
            }
            __syncthreads();
            if (sm.last) {
                auto part_of = [&](int c) { return parts + (2 * c + (c == c0 ? 1 : 0)) * static_cast<long long>(kPart); };
                for (int x = 4 * tid; x < n_rows * DP; x += 4 * kThreads) {
                    const int r = x / DP;
                    float mx = -INFINITY;
                    for (int c = c0; c <= c1; c++) mx = fmaxf(mx, __ldcg(part_of(c) + kRows * DP + r));
                    float sum = 0.0f;
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (int c = c0; c <= c1; c++) {
                        const float *q = part_of(c);
                        const float mc = __ldcg(q + kRows * DP + r);
                        const float4 u = __ldcg(reinterpret_cast<const float4 *>(q + x));
                        if (mc == -INFINITY) continue;
                        const float k = exp2f(mc - mx);
                        sum = fmaf(k, __ldcg(q + kRows * DP + kRows + r), sum);
                        v.x = fmaf(k, u.x, v.x);
                        v.y = fmaf(k, u.y, v.y);
                        v.z = fmaf(k, u.z, v.z);
                        v.w = fmaf(k, u.w, v.w);
                    }
                    const float inv = mx == -INFINITY ? 0.0f : 1.0f / sum;
                    put(r, x - r * DP, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                }
            }
        }

        // ---- on to the next item ----
        pos += ITEMS ? static_cast<int>(gridDim.x) : n_slots;
        off = 0;
        if (pos < end) {
            if (!ITEMS) {
                item++;
                if (item == work.tiles * p.c.heads) {
                    item = 0;
                    do {
                        seq++;
                        work = work_of<kRows>(p, group, seq);
                    } while (work.slots == 0);
                }
            }
            fence_proxy_async_smem();  // the sums were read and written as plain memory, TMA writes there next
            __syncthreads();
        }
    }
}

// Tiles of 8 rows per CTA. More rows than a CTA takes become row tiles that
// each read the cache.
int tiles_of(const Cache &c, int max_new, int q_heads) {
    const long long rows = (long long)max_new * (q_heads / c.heads);
    return rows <= 8 ? 1 : 2;
}

// What the beginning and end of an item and of a part cost, in the time a warp
// takes for a pair of blocks, about 1 us (measured: 1024 items of 11 blocks
// 19.7 us whole, 33.5 us divided; 512 of 66 blocks 39 and 44 us; 8 of 250
// blocks 32 and 21 us).
constexpr long long kItemCost = 3, kPartCost = 8;

template <int DP, int NT, bool SPLIT, bool ITEMS>
cudaError_t launch3(const AttendParams &p, const CUtensorMap &k_map, const CUtensorMap &v_map, long long grid, cudaStream_t s) {
    constexpr int kBytes = Layout<DP, NT, SPLIT>::kBytes;
    auto kernel = p.c.fp8 ? k_attend<DP, NT, SPLIT, true, ITEMS> : k_attend<DP, NT, SPLIT, false, ITEMS>;
    static SmemOptIn opt_in[2];
    const cudaError_t e = opt_in[p.c.fp8].set(reinterpret_cast<const void *>(kernel), kBytes);
    if (e != cudaSuccess) return e;
    kernel<<<(unsigned)grid, kThreads, kBytes, s>>>(k_map, v_map, p);
    return cudaGetLastError();
}

template <int DP, int NT, bool SPLIT>
cudaError_t launch2(const AttendParams &p, int sms, cudaStream_t s) {
    CUtensorMap k_map, v_map;
    if (!codes_map(&k_map, p.c, p.c.k, DP, kBlk) || !codes_map(&v_map, p.c, p.c.v, DP, kBlk)) return cudaErrorInvalidValue;
    // one wave; fewer CTAs when there are not kMinBlocks for each
    const long long rows = (long long)p.b.max_new * (p.q.heads / p.c.heads), tiles = (rows + 8 * NT - 1) / (8 * NT);
    const long long items = (long long)p.b.n_seqs * p.c.heads * tiles;
    long long seen = p.b.max_len;
    if (p.window) seen = std::min<long long>(seen, (long long)p.window + p.sinks + p.b.max_new + kBlk);
    const long long blocks = seen / kBlk + 2, wave = (long long)sms * ctas_per_sm<NT, SPLIT>();
    // the longest item's pairs decide how long whole items take; an even
    // division over CTAs pays for the beginning and end of each part
    const long long pairs = (blocks + 1) / 2;
    const long long whole = (items + wave - 1) / wave * ((pairs + kWarps - 1) / kWarps + kItemCost);
    const long long even = items * pairs / (kWarps * wave) + kPartCost * (items / wave + 2);
    if (tiles == 1 && whole <= even) return launch3<DP, NT, SPLIT, true>(p, k_map, v_map, std::min(wave, items), s);
    const long long most = std::min<long long>(items * ((blocks + kMinBlocks - 1) / kMinBlocks), kCounters);
    return launch3<DP, NT, SPLIT, false>(p, k_map, v_map, std::min(wave, most), s);
}

template <int DP>
cudaError_t launch1(const AttendParams &p, int nt, bool split_f32, int sms, cudaStream_t s) {
    if (split_f32) return nt == 1 ? launch2<DP, 1, true>(p, sms, s) : launch2<DP, 2, true>(p, sms, s);
    return nt == 1 ? launch2<DP, 1, false>(p, sms, s) : launch2<DP, 2, false>(p, sms, s);
}

}  // namespace

size_t attend_workspace(const Cache &c, const Batch &b, int q_heads, int sms) {
    const int nt = tiles_of(c, b.max_new, q_heads);
    const size_t ctas = std::min<size_t>((size_t)sms * (nt == 1 ? ctas_per_sm<1, false>() : ctas_per_sm<2, false>()), kCounters);
    const size_t floats = ctas * 2 * (8 * nt) * ((c.dim <= 64 ? 64 : 128) + 2);
    return kCounters * sizeof(int) + floats * sizeof(float);
}

cudaError_t attend(const AttendParams &p, int sms, cudaStream_t s) {
    const bool split_f32 = p.out.dtype == kF32;
    const int nt = tiles_of(p.c, p.b.max_new, p.q.heads);
    if (!split_f32 && nt > 1 && p.b.n_seqs <= kTiledSeqs) {
        // Many rows: a tile of 64 keys takes the tiled kernel about 0.8 us for 256 rows, an SM at a time;
        // here the GPU takes about 1200 blocks of 16 keys by 16 rows a microsecond, wherever they are.
        const long long rows = (long long)p.b.max_new * (p.q.heads / p.c.heads);
        long long seen = p.b.max_len;
        if (p.window) seen = std::min<long long>(seen, (long long)p.window + p.sinks + p.b.max_new);
        const double here = (double)p.b.n_seqs * p.c.heads * ((rows + 15) / 16) * (seen / kBlk + 1) / 1200.0;
        if (rows > 16 && 0.8 * tiled_rounds(p, sms, seen) < here) return attend_tiled(p, s);
    }
    return p.c.dim <= 64 ? launch1<64>(p, nt, split_f32, sms, s) : launch1<128>(p, nt, split_f32, sms, s);
}

}  // namespace kv
}  // namespace ditch
