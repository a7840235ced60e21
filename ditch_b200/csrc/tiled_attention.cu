// Causal attention with a sliding window and sinks on the fifth-generation
// tensor cores, for many query rows: over contiguous f16 / bf16 rows, and over
// the paged 8-bit cache.
//
// Bound by the tensor cores and, just as much, by the exponentials: 128 x 128
// scores take 512 cycles of MMA for Q.K^T, 512 for P.V (head size 128) and
// 1024 cycles of the SFU. Two row tiles of 128 query rows are on an SM, whose
// products and softmax alternate, in one CTA or in two:
//   first warps      softmax, four warps a row tile, a row a thread
//   then one         issues the MMAs
//   then one         loads by TMA (contiguous rows), or looks up the pages and
//                    scales of the tiles to come (the cache)
//   warps 12-15      turn 8-bit codes into f16 operands (the cache)
// A row tile is all the query heads of one key / value head for as many
// tokens as fill 128 rows, so that a window or the causal limit cuts as close
// as a few tokens, and two tiles of one CTA read the same keys and values.
//
// TMEM: for each row tile S (128 columns: one tile of 128 keys, or two of 64)
// and O (128). P goes back over its S as 16-bit pairs and is the A operand of
// P.V from there; V is taken as it lies, [token][dimension], as a transposed
// (MN-major) B operand. Three shapes (Shape), by measurement at head size 128:
//   128 keys, two row tiles a CTA: the least MMA time, for long runs of keys
//     (8192 tokens, window 4096: 838 us in a steady loop, which meets the
//     power limit, and 744 us in bursts of three; with 64 keys 955 and 912 us,
//     in one row tile a CTA 932 and 825 us: an MMA with N = 64 takes the 64
//     cycles of one with N = 128, for its A operand)
//   64 keys, two row tiles: S(j + 1) is made while the softmax works on S(j);
//     for the cache, whose codes then need half the registers on their way
//     (4 sequences of 512 rows over 2500 to 6000: 238 us against 307 us, when
//     it was chosen)
//   64 keys, one row tile, two CTAs an SM: short runs, where the beginning
//     and end of a CTA count
// Measured: 8192 rows of 64 heads under a window of 4096 in 729 to 744 us in
// bursts, 1110 to 1130 TFLOP/s (0.66 to 0.68 of the burst peak of a plain
// product), 830 to 859 us in a loop, 961 to 995 TFLOP/s (0.69 to 0.71 of the
// sustained peak); 4 x 512 rows over the cache in 217 to 222 us, 550 TFLOP/s.
// Taking 25 to 50 % of the exponentials off the SFU (a polynomial on the FMA
// pipe) changed nothing or cost 2 to 11 %.
//
// A row whose maximum has grown by more than 2^kLazy since its sums'
// reference rescales its part of O in TMEM, once P.V(j - 1) is in; most never
// do.
//
// The cache's codes are f16 operands exactly (int8 and E4M3 fit), laid out in
// shared memory as TMA would; Q is brought into f16's range by a power of two
// for each row and rounded to it (f32 queries to 11 bits: a second half would
// take the shared memory of a row tile and a third of the MMAs again). A block's scales work on the scores: sk in the factor that
// multiplies them, sv, as a fraction of the largest in sight, in the exponent
// of the weight that goes into P (taken out again of the sum of weights). A
// row's reference maximum is that of the scores with it, so the largest of the
// weights that go into P is about 1, however small the values that the row
// sees are beside others.
//
// What a row does not see has weight 0 in the product, and 0 times an
// infinity or NaN is NaN: rows whose result is not finite are computed again
// from the keys that they do see (compute_row). A scale of the cache that is
// not finite stays out of the products, and makes the rows that see it NaN.
//
// Contiguous rows that TMA cannot take (not 16-byte aligned) go by
// k_window_rows, one warp for each row.
#include <algorithm>

#include "attn_common.cuh"
#include "gemm.cuh"
#include "kv_range.cuh"

namespace ditch {
namespace kv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.0f;   // a weight stays below 2^8 of the reference
constexpr float kF16Up = 7.0f;  // and is taken times 2^7 where P is f16: its normal numbers then reach down to 2^-21
constexpr int kRowWarps = 4;

// ---- one row by one warp -----------------------------------------------------------
// Lane l holds dimensions 4 l .. 4 l + 3 of the head.
struct RowState {
    float m = -INFINITY, sum = 0.0f, o[4] = {0, 0, 0, 0};
    __device__ void key(const float (&q)[4], const float (&k)[4], const float (&v)[4], float scale2) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) s = fmaf(q[i], k[i], s);
        s = attn::warp_sum(s) * scale2;
        const float top = fmaxf(m, s);  // (of a NaN and a number, the number)
        const float keep = top == -INFINITY ? 1.0f : exp2f(m - top);
        const float w = s == -INFINITY ? 0.0f : exp2f(s - top);  // a NaN score is a NaN weight, also while there is no maximum
        m = top;
        sum = sum * keep + w;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = o[i] * keep + w * v[i];
    }
};

__device__ __forceinline__ int next_key(int j, int p, int window, int sinks) {
    j++;
    return window && j >= sinks && j <= p - window ? p - window + 1 : j;
}

__device__ __forceinline__ int first_key(int p, int window, int sinks) {
    return window && sinks == 0 && p >= window ? p - window + 1 : 0;
}

// Where keys and values come from.
struct Contiguous {
    Rows k, v;
    const int32_t *ko;
    int n_kv, max_kv;
};

struct Paged {
    Cache c;
    Batch b;
};

struct TiledParams {
    Rows q, out;
    const int32_t *qo;
    int n_seqs, n_q, max_q, kv_heads, dim;
    float scale;
    int window, sinks;
    int *status;
    Contiguous rows;
    Paged paged;
};

// Sequence `seq`: its query rows and keys (k0: its first key's row), none
// (and the status word set) when the device's numbers leave the host's bounds.
struct Seq {
    int q0, nq, k0, nk;
};

template <bool PAGED>
__device__ __forceinline__ Seq seq_of(const TiledParams &p, int seq) {
    Seq s;
    if (PAGED) {
        const Span a = span_of(p.paged.b, p.paged.c.page_shift, seq, p.status);
        s.q0 = a.row0, s.nq = a.n, s.k0 = 0, s.nk = a.len;
        return s;
    }
    s.q0 = __ldg(p.qo + seq);
    s.k0 = __ldg(p.rows.ko + seq);
    const int q1 = __ldg(p.qo + seq + 1), k1 = __ldg(p.rows.ko + seq + 1);
    s.nq = q1 - s.q0;
    s.nk = k1 - s.k0;
    if (s.q0 < 0 || q1 > p.n_q || s.nq < 0 || s.nq > p.max_q || s.k0 < 0 || k1 > p.rows.n_kv || s.nk < 0 || s.nk > p.rows.max_kv) {
        flag(p.status);
        s.nq = s.nk = 0;
    }
    return s;
}

// Query row `tok` of head `head`, at position pos of sequence `seq`, whose
// contiguous keys begin at row k0.
template <bool PAGED>
__device__ __noinline__ void compute_row(const TiledParams &p, int seq, int tok, int head, int pos, int k0, int lane) {
    const int d = 4 * lane, kvh = head / (p.q.heads / p.kv_heads);
    float q[4] = {0, 0, 0, 0};
    for (int e = 0; e < 4; e++)
        if (d + e < p.dim) q[e] = load1(p.q, tok * p.q.ts + head * p.q.hs + d + e);
    RowState st;
    for (int j = first_key(pos, p.window, p.sinks); j <= pos; j = next_key(j, pos, p.window, p.sinks)) {
        float k[4] = {0, 0, 0, 0}, v[4] = {0, 0, 0, 0};
        if (PAGED) {
            const Cache &c = p.paged.c;
            const int page = page_of(c, p.paged.b, seq, j, p.status);
            if (page < 0) continue;
            if (d < p.dim) {
                const long long at = code_at(c, page, kvh, j) + d, sa = scale_at(c, page, kvh, j);
                decode4(c.fp8, *reinterpret_cast<const uint32_t *>(c.k + at), k);
                decode4(c.fp8, *reinterpret_cast<const uint32_t *>(c.v + at), v);
                for (int e = 0; e < 4; e++) {
                    k[e] *= c.ks[sa];
                    v[e] *= c.vs[sa];
                }
            }
        } else {
            for (int e = 0; e < 4; e++)
                if (d + e < p.dim) {
                    k[e] = load1(p.rows.k, (k0 + j) * p.rows.k.ts + kvh * p.rows.k.hs + d + e);
                    v[e] = load1(p.rows.v, (k0 + j) * p.rows.v.ts + kvh * p.rows.v.hs + d + e);
                }
        }
        st.key(q, k, v, p.scale * kLog2e);
    }
    for (int e = 0; e < 4; e++)
        if (d + e < p.dim) store1(p.out, tok * p.out.ts + head * p.out.hs + d + e, st.m == -INFINITY && st.sum == 0.0f ? 0.0f : st.o[e] / st.sum);
}

__global__ void __launch_bounds__(kRowWarps * 32) k_window_rows(TiledParams p) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long row = static_cast<long long>(blockIdx.x) * kRowWarps + warp;
    if (row >= static_cast<long long>(p.n_q) * p.q.heads) return;
    const int tok = static_cast<int>(row / p.q.heads), head = static_cast<int>(row % p.q.heads);
    int seq = 0;
    while (seq + 1 < p.n_seqs && __ldg(p.qo + seq + 1) <= tok) seq++;
    const Seq s = seq_of<false>(p, seq);
    if (tok < s.q0 || tok >= s.q0 + s.nq) return;
    compute_row<false>(p, seq, tok, head, s.nk - s.nq + tok - s.q0, s.k0, lane);
}

// ---- the tiled kernel ------------------------------------------------------------------
constexpr int kTileRows = 128;  // query rows of a tile: the MMA's M, a TMEM lane each

constexpr int kConverters = 128;  // threads that turn codes into operands

// KEYS: of a tile; TILES: row tiles of a CTA.
template <bool PAGED_, int KEYS_, int TILES_>
struct Shape {
    static constexpr bool kPaged = PAGED_;
    static constexpr int kKeys = KEYS_, kTiles = TILES_;
    static constexpr int kBuffers = 128 / KEYS_;                       // of S, a row tile
    static constexpr int kStages = KEYS_ == 128 || TILES_ == 1 ? 2 : 4;  // tiles of K and of V in shared memory
    // Registers that the softmax warps take from the others at the start (setmaxnreg; 512 threads begin with 128
    // each, 384 with 168): they hold a row of scores. With 64 keys and no converters, what they begin with is enough.
    static constexpr bool kTrade = PAGED_ || KEYS_ == 128;
    static constexpr int kThreads = PAGED_ ? 384 + kConverters : kTrade ? 384 : 128 * TILES_ + 64;
    static constexpr int kSoftmaxRegs = PAGED_ ? 160 : 208, kIssueRegs = 80, kConvertRegs = 112;
    static constexpr int kCtas = TILES_ == 1 ? 2 : 1;                  // an SM
    static constexpr int kIssuer = 4 * TILES_, kLoader = kIssuer + 1;  // warps
    static constexpr uint32_t kTmem = 256 * TILES_;
};
constexpr int kScaleSlots = 8;    // tiles whose pages and scales are known at a time

template <int DP, class S>
struct Layout {
    static constexpr int kQHalf = kTileRows * 128, kKHalf = S::kKeys * 128;  // 64 dimensions of a tile's rows
    static constexpr int kQTile = kQHalf * (DP / 64), kKTile = kKHalf * (DP / 64);
    static constexpr int kBytes = 1024 + S::kTiles * kQTile + 2 * S::kStages * kKTile;
};

constexpr int kMostStages = 4, kScaleKeys = 64;  // (the cache's tiles are of 64 keys)

struct Bars {
    uint64_t q_full, k_full[kMostStages], k_empty[kMostStages], v_full[kMostStages], v_empty[kMostStages];
    uint64_t s_full[2][2], p_full[2][2],  // P of the two tiles of 64 keys, or of the two halves of 128
         o_full[2], scales_full[kScaleSlots], scales_empty[kScaleSlots];
    // per 16 keys of a tile: the factor of scores, log2 of sv / the largest sv, its inverse
    // and the offsets of their K and V codes (-1: zeros)
    long long codes[2][kScaleSlots][kScaleKeys / 16];
    float sk[kScaleSlots][kScaleKeys / 16], lv[kScaleSlots][kScaleKeys / 16], iv[kScaleSlots][kScaleKeys / 16];
    uint32_t bad[kScaleSlots];  // a byte for each 16 keys: a scale is not finite
    float v_top;                // the largest finite sv in sight
    uint32_t tmem;
    int abort;
};

template <int N>
__device__ __forceinline__ void give_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <int N>
__device__ __forceinline__ void take_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// Shared-memory descriptor of an MN-major operand with 128-byte swizzle, rows
// of 64 elements for each k: 8 rows are an atom of 1024 bytes (SBO between
// atoms along k), the next 64 elements of the operand's rows LBO further on.
__device__ __forceinline__ uint64_t sw128_mnmajor_desc(uint32_t smem_addr, uint32_t lbo) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3fff);
    d |= static_cast<uint64_t>((lbo >> 4) & 0x3fff) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

// kind::f16 with f32 accumulation: type 0 = f16, 1 = bf16; b_mn: B is MN-major.
__device__ __forceinline__ uint32_t idesc_of(uint32_t type, bool b_mn, int n) {
    return (1u << 4) | (type << 7) | (type << 10) | (b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(kTileRows >> 4) << 24);
}

// D += A[tmem] * B[smem]
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// One lane of a converged warp. The issuing warp runs its loop as a whole, so
// that descriptors stay in uniform registers, and only the MMAs are this
// lane's: in a loop of one lane every MMA took about 100 cycles to issue.
__device__ __forceinline__ bool elect_one() {
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}

__device__ __forceinline__ void tma_load_rows(const CUtensorMap *map, uint64_t *bar, void *dst, int d, int head, int row) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(d), "r"(head), "r"(row)
        : "memory");
}

// 32 columns of this thread's TMEM lane, without waiting ...
__device__ __forceinline__ void tmem_ld32_start(uint32_t at, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}

// ... and the point after which the registers may be used.
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
        "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
        "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void tmem_st16_start(uint32_t at, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float exp2_sfu(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Two f32 in a 64-bit register, for the packed arithmetic.
using f32x2 = unsigned long long;

__device__ __forceinline__ f32x2 pair_of(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float2 floats_of(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}

__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    if (BF16) return pack_bf16x2(lo, hi);
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// A row tile holds `heads` query heads of one key / value head (chunk of them
// when a group has more than 128) for `toks` tokens: row = token * heads + head.
struct Tiling {
    int heads, toks, chunks;
};

// Sixteen codes (dimensions 16 c ... of key r) as two 16-byte pieces of the
// f16 operand tile, where TMA would have put them.
template <bool FP8>
__device__ __forceinline__ void put_codes(uint8_t *tile, int half_bytes, int r, int c, uint4 u) {
    uint32_t w[8];
    const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (FP8) {
            e4m3_pairs(x[i], w[2 * i], w[2 * i + 1]);
        } else {
            const uint32_t b = x[i] ^ 0x80808080u;
            w[2 * i] = int8_pair(b, 0x4140);
            w[2 * i + 1] = int8_pair(b, 0x4342);
        }
    }
    uint8_t *row = tile + (c >> 2) * half_bytes + r * 128;
    const int a = 2 * (c & 3), sw = r & 7;
    // the two halves' lanes store their pieces in opposite order, so that eight lanes cover all banks
    const bool flip = c >> 2;
    const uint4 p0 = make_uint4(w[0], w[1], w[2], w[3]), p1 = make_uint4(w[4], w[5], w[6], w[7]);
    *reinterpret_cast<uint4 *>(row + (((flip ? a + 1 : a) ^ sw) << 4)) = flip ? p1 : p0;
    *reinterpret_cast<uint4 *>(row + (((flip ? a : a + 1) ^ sw) << 4)) = flip ? p0 : p1;
}

// BF16: the type of out (and of contiguous operands); the cache's operands are f16.
template <int DP, bool BF16, bool FP8, class S>
__global__ void __launch_bounds__(S::kThreads, S::kCtas)
    k_tiled(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
            const __grid_constant__ CUtensorMap v_map, TiledParams p, Tiling tl, int pairs) {
    using L = Layout<DP, S>;
    constexpr bool PAGED = S::kPaged;
    constexpr int kTileKeys = S::kKeys, kStages = S::kStages, kBuffers = S::kBuffers;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Bars bars;
    // the longest runs of keys first: the longest sequences (where there are few), and their last rows
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int pair = pairs - 1 - blockIdx.x / (tl.chunks * p.kv_heads);
    int x = blockIdx.x % (tl.chunks * p.kv_heads), seq = blockIdx.y;
    if (p.n_seqs <= 32 && p.n_seqs > 1) {
        int len = -1;
        if (lane < p.n_seqs) len = PAGED ? __ldg(p.paged.b.lens + lane) : __ldg(p.rows.ko + lane + 1) - __ldg(p.rows.ko + lane);
        int before = 0;
        for (int i = 0; i < p.n_seqs; i++) {
            const int other = __shfl_sync(0xffffffffu, len, i);
            before += other > len || (other == len && i < lane);
        }
        seq = __ffs(__ballot_sync(0xffffffffu, lane < p.n_seqs && before == static_cast<int>(blockIdx.y))) - 1;
    }
    const int chunk = x % tl.chunks, kvh = x / tl.chunks;
    const Seq sq = seq_of<PAGED>(p, seq);
    const int i0 = pair * S::kTiles * tl.toks;  // first token of the CTA's
    if (i0 >= sq.nq) return;
    const int tiles = S::kTiles == 2 && i0 + tl.toks < sq.nq ? 2 : 1;
    const int group = p.q.heads / p.kv_heads;
    const int first = sq.nk - sq.nq;  // position of the sequence's first query
    const int p_lo = first + i0, p_hi = first + min(sq.nq, i0 + S::kTiles * tl.toks) - 1;
    Range range = range_of(max(p_lo, 0), max(p_hi, 0), p.window, p.sinks, kTileKeys);
    const int n = p_hi < 0 ? 0 : range.n;
    auto keys_of = [&](int j) {  // of tile j: up to the last row's position, in whole MMA steps
        return min(kTileKeys, (p_hi + 1 - range.token(j, kTileKeys) + 15) & ~15);
    };

    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *s_q = base, *s_k = base + S::kTiles * L::kQTile, *s_v = s_k + kStages * L::kKTile;
    // Contiguous rows: Q, and K (kv 0) or V (kv 1) of tile j.
    auto load = [&](int kv, int j) {
        uint64_t *full = kv ? &bars.v_full[j % kStages] : &bars.k_full[j % kStages];
        mbar_arrive_expect_tx(full, L::kKTile);
        uint8_t *dst = (kv ? s_v : s_k) + j % kStages * L::kKTile;
#pragma unroll
        for (int h = 0; h < DP / 64; h++)
            tma_load_rows(kv ? &v_map : &k_map, full, dst + h * L::kKHalf, 64 * h, kvh, sq.k0 + range.token(j, kTileKeys));
    };
    auto load_first = [&]() {
        const int head0 = kvh * group + chunk * tl.heads;
        mbar_arrive_expect_tx(&bars.q_full, tiles * (DP / 64) * tl.heads * tl.toks * 128);
        for (int t = 0; t < tiles; t++)
#pragma unroll
            for (int h = 0; h < DP / 64; h++)
                tma_load_rows(&q_map, &bars.q_full, s_q + t * L::kQTile + h * L::kQHalf, 64 * h, head0, sq.q0 + i0 + t * tl.toks);
        for (int j = 0; j < min(n, kStages); j++) {
            load(0, j);
            load(1, j);
        }
    };
    if (warp == S::kLoader && lane == 0) {
        if (!PAGED) {
            tma_prefetch_desc(&q_map);
            tma_prefetch_desc(&k_map);
            tma_prefetch_desc(&v_map);
        }
        mbar_init(&bars.q_full, PAGED ? tiles * kTileRows : 1);
        for (int i = 0; i < kStages; i++) {
            mbar_init(&bars.k_full[i], PAGED ? kConverters : 1);
            mbar_init(&bars.k_empty[i], 1);
            mbar_init(&bars.v_full[i], PAGED ? kConverters : 1);
            mbar_init(&bars.v_empty[i], 1);
        }
        for (int i = 0; i < S::kTiles; i++) {
            for (int b = 0; b < kBuffers; b++) {
                mbar_init(&bars.s_full[i][b], 1);
            }
            for (int b = 0; b < 2; b++) mbar_init(&bars.p_full[i][b], kTileRows);
            mbar_init(&bars.o_full[i], 1);
        }
        for (int i = 0; i < kScaleSlots; i++) {
            mbar_init(&bars.scales_full[i], kScaleKeys / 16);
            mbar_init(&bars.scales_empty[i], 1);
        }
        bars.abort = 0;
        fence_barrier_init();
        if (!PAGED && n > 0) load_first();
    }
    if (warp == S::kIssuer) {
        tmem_alloc(&bars.tmem, S::kTmem);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars.tmem;
    int *status = p.status;
    volatile int *abort = &bars.abort;

    if (S::kTrade && warp >= 8 && warp < 12) give_registers<S::kIssueRegs>();
    if (PAGED && warp >= 12) {
        give_registers<S::kConvertRegs>();
        if (n > 0) {
            // ---- codes to operands ----
            const Cache &c = p.paged.c;
            const int me = tid - 384;
            constexpr int kChunks = DP / 16;                             // 16-byte pieces of a key's codes
            constexpr int kMine = kTileKeys * kChunks / kConverters;     // of a thread, for a tile
            const int chunk16 = me % kChunks, r0 = me / kChunks;         // its keys are r0 + i * kConverters / kChunks
            // unit u: K (even) or V (odd) of tile u / 2
            const bool in = 16 * chunk16 < c.dim;
            bool live = true;
            uint4 buf[2][kMine];
            auto fetch = [&](int u, uint4(&x)[kMine]) {
                if (u >= 2 * n) return;
                const int j = u >> 1, slot = j % kScaleSlots;
                if (!(u & 1) && live) live = mbar_wait(&bars.scales_full[slot], (j / kScaleSlots) & 1, abort, status);
                if (!live) return;
                const uint8_t *codes = (u & 1 ? c.v : c.k) + (r0 & 15) * c.dim + 16 * chunk16;
                const int last = p_hi - range.token(j, kTileKeys) - r0;
#pragma unroll
                for (int i = 0; i < kMine; i++) {
                    const int at = i * (kConverters / kChunks);
                    const long long off = bars.codes[u & 1][slot][(r0 + at) >> 4];
                    x[i] = at <= last && off >= 0 && in ? __ldg(reinterpret_cast<const uint4 *>(codes + off)) : make_uint4(0, 0, 0, 0);
                }
            };
            auto put = [&](int u, const uint4(&x)[kMine]) {
                const int j = u >> 1, st = j % kStages;
                const bool value = u & 1;
                if (!live) return false;
                if (j >= kStages && !mbar_wait(value ? &bars.v_empty[st] : &bars.k_empty[st], (j / kStages + 1) & 1, abort, status)) return false;
                uint8_t *dst = (value ? s_v : s_k) + st * L::kKTile;
#pragma unroll
                for (int i = 0; i < kMine; i++) put_codes<FP8>(dst, L::kKHalf, r0 + i * (kConverters / kChunks), chunk16, x[i]);
                fence_proxy_async_smem();
                mbar_arrive(value ? &bars.v_full[st] : &bars.k_full[st]);
                return true;
            };
            fetch(0, buf[0]);
            for (int u = 0; u < 2 * n; u += 2) {
                fetch(u + 1, buf[1]);
                if (!put(u, buf[0])) break;
                fetch(u + 2, buf[0]);
                if (!put(u + 1, buf[1])) break;
            }
        }
    } else if (PAGED && warp == S::kLoader) {
        if (n > 0) {
            // ---- pages and scales ----
            const Cache &c = p.paged.c;
            // the largest finite sv in sight and the smallest that is not 0 (as bits)
            const int per_tile = kTileKeys >> c.block_shift;
            // A tile can hold pages of which no row sees a key (before the window, after the sinks): they may be anyone's,
            // or nobody's, and are not looked up. Their keys are hidden from all rows, whatever stands for them.
            auto in_sight = [&](int key, int keys) { return key <= p_hi && (!p.window || key + keys > p_lo - p.window + 1 || key < p.sinks); };
            uint32_t top = 0, least = 0x7f800000u;
            for (int b = lane; b < n * per_tile; b += 32) {
                const int key = range.token(b / per_tile, kTileKeys) + ((b % per_tile) << c.block_shift);
                if (!in_sight(key, 1 << c.block_shift)) continue;
                const int page = page_of(c, p.paged.b, seq, key, p.status);
                const uint32_t sv = page >= 0 ? __float_as_uint(__ldg(c.vs + scale_at(c, page, kvh, key))) & 0x7fffffffu : 0u;
                if (sv < 0x7f800000u) {
                    top = max(top, sv);
                    if (sv) least = min(least, sv);
                }
            }
            top = __reduce_max_sync(0xffffffffu, top);
            least = __reduce_min_sync(0xffffffffu, least);
            const float v_top = top ? __uint_as_float(top) : 1.0f;
            if (lane == 0) bars.v_top = v_top;
            // Ratios down to 2^-100 leave every weight that counts above 2^-126, where exp2 gives 0. Values that are all 0
            // (their codes then count as 0) go by the smallest sv, so that their weights are in the others' reach.
            constexpr float kLeast = 0x1p-100f;
            const float nil = top ? fmaxf(__uint_as_float(least) / v_top, kLeast) : 1.0f;
            // a lane for each 16 keys of eight tiles, so that the loads' latencies are paid once for all of them
            static_assert(kScaleSlots * (kScaleKeys / 16) == 32, "a lane each");
            const int block = lane % (kScaleKeys / 16);
            for (int j = lane / (kScaleKeys / 16); j < n; j += kScaleSlots) {
                const int key = range.token(j, kTileKeys) + 16 * block, slot = j % kScaleSlots;
                float sk = 0.0f, sv = 0.0f;
                long long codes = -1;
                bool bad = false;
                if (in_sight(key, 16)) {
                    const int page = page_of(c, p.paged.b, seq, key, p.status);
                    sk = __uint_as_float(0x7fc00000u);  // no page: the row is computed again without it
                    if (page >= 0) {
                        const long long at = scale_at(c, page, kvh, key);
                        codes = code_at(c, page, kvh, key);
                        sk = __ldg(c.ks + at);
                        sv = __ldg(c.vs + at);
                        bad = !(fabsf(sk) <= 3.4e38f && fabsf(sv) <= 3.4e38f);
                        if (bad) sk = sv = 0.0f;  // for the rows that do not see it
                    }
                }
                float ratio = sv == 0.0f ? nil : sv / v_top;
                if (!(ratio >= kLeast)) ratio = __uint_as_float(0x7fc00000u);  // the rows are computed again, one at a time
                if (j >= kScaleSlots && !mbar_wait(&bars.scales_empty[slot], (j / kScaleSlots + 1) & 1, abort, status)) break;
                bars.codes[0][slot][block] = codes;
                bars.codes[1][slot][block] = sv == 0.0f ? -1 : codes;
                bars.sk[slot][block] = sk == 0.0f ? 0x1p-100f : sk;  // never 0: a hidden score of -inf stays one
                reinterpret_cast<uint8_t *>(&bars.bad[slot])[block] = bad;
                bars.lv[slot][block] = log2f(ratio);
                bars.iv[slot][block] = 1.0f / ratio;
                mbar_arrive(&bars.scales_full[slot]);
            }
        }
    } else if (warp == S::kLoader) {
        if (lane == 0 && n > 0) {
            bool go = true;
            for (int j = kStages; go && j < n; j++)
                for (int kv = 0; go && kv < 2; kv++) {
                    go = mbar_wait(kv ? &bars.v_empty[j % kStages] : &bars.k_empty[j % kStages], (j / kStages + 1) & 1, abort, status);
                    if (go) load(kv, j);
                }
        }
    } else if (warp == S::kIssuer) {
        if (n > 0) {
            constexpr uint32_t kType = BF16 && !PAGED ? 1 : 0;
            const bool leader = elect_one();
            const uint32_t q_at = smem_u32(s_q), k_at = smem_u32(s_k), v_at = smem_u32(s_v);
            auto qk = [&](int t, int j) {
                const uint32_t id = idesc_of(kType, false, keys_of(j));
                const uint64_t a = sw128_kmajor_desc(q_at + t * L::kQTile), b = sw128_kmajor_desc(k_at + (j % kStages) * L::kKTile);
                const uint32_t d = tmem + 128 * t + kTileKeys * (j % kBuffers);
                if (leader) {
#pragma unroll
                    for (int h = 0; h < DP / 64; h++)
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            tc_mma_bf16(d, a + (h * L::kQHalf >> 4) + 2 * k, b + (h * L::kKHalf >> 4) + 2 * k, id, (h | k) ? 1u : 0u);
                    tc_commit(&bars.s_full[t][j % kBuffers]);
                    if (t == tiles - 1) tc_commit(&bars.k_empty[j % kStages]);
                }
                __syncwarp();
            };
            bool ok = mbar_wait_warp(&bars.q_full, 0, abort, status);
            for (int j = 0; ok && j < min(kBuffers, n); j++) {
                ok = mbar_wait_warp(&bars.k_full[j], 0, abort, status);
                if (!ok) break;
                tc_fence_after();
                for (int t = 0; t < tiles; t++) qk(t, j);
            }
            // what the products of step j read besides P: V(j) and K(j + kBuffers)
            auto operands = [&](int j) {
                return mbar_wait_warp(&bars.v_full[j % kStages], (j / kStages) & 1, abort, status) &&
                       (j + kBuffers >= n ||
                        mbar_wait_warp(&bars.k_full[(j + kBuffers) % kStages], ((j + kBuffers) / kStages) & 1, abort, status));
            };
            ok = ok && operands(0);
            for (int j = 0; ok && j < n; j++) {
                const int st = j % kStages, steps = keys_of(j) / 16;
                for (int t = 0; ok && t < tiles; t++) {
                    const uint32_t id = idesc_of(kType, true, DP), d = tmem + 128 * (S::kTiles + t), a = tmem + 128 * t + kTileKeys * (j % kBuffers);
                    const uint64_t v = sw128_mnmajor_desc(v_at + st * L::kKTile, L::kKHalf);
#pragma unroll
                    for (int half = 0; half < kTileKeys / 64; half++) {
                        if (!ok) break;
                        ok = mbar_wait_warp(&bars.p_full[t][kBuffers == 2 ? j & 1 : half], (j / kBuffers) & 1, abort, status);
                        if (!ok) break;
                        tc_fence_after();
                        if (leader) {
#pragma unroll
                            for (int k = 4 * half; k < 4 * half + 4; k++)
                                if (k < steps) tc_mma_ts(d, a + 8 * k, v + k * (16 * 128 >> 4), id, (j | k) ? 1u : 0u);
                        }
                        __syncwarp();
                    }
                    if (!ok) break;
                    if (leader) {
                        if (t == tiles - 1) tc_commit(&bars.v_empty[st]);
                        if (PAGED && t == tiles - 1) tc_commit(&bars.scales_empty[j % kScaleSlots]);
                        if (j + 1 == n) tc_commit(&bars.o_full[t]);
                    }
                    __syncwarp();
                    if (j + kBuffers < n) qk(t, j + kBuffers);
                }
                if (ok && j + 1 < n) ok = operands(j + 1);  // while the MMAs are under way
            }
        }
    } else if (warp < 4 * S::kTiles) {
        if (S::kTrade) take_registers<S::kSoftmaxRegs>();
        if ((warp >> 2) < tiles) {
            // ---- softmax of tile t: this thread's row ----
            const int t = warp >> 2, row = tid & 127;
            const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
            const uint32_t s_cols = tmem + lanes + 128 * t, o_at = tmem + lanes + 128 * (S::kTiles + t);
            const int tok = row / tl.heads, head = row - tok * tl.heads;  // of the tile
            const int i = i0 + t * tl.toks + tok, pos = first + i;
            const bool valid = tok < tl.toks && i < sq.nq && chunk * tl.heads + head < group;
            // the tile's rows: the tiles of keys that all of them see whole need no masks
            const int t_lo = first + i0 + t * tl.toks, t_hi = min(t_lo + tl.toks, first + sq.nq) - 1;
            float c = p.scale * kLog2e;
            if (PAGED && n > 0) {
                // Q to f16: the row by a power of two to below 2, which c makes good
                const int h = kvh * group + chunk * tl.heads + head;
                const long long at = (sq.q0 + i) * p.q.ts + h * p.q.hs;
                uint32_t top = 0;
                if (valid)
                    for (int d = 0; d < p.dim; d += 4) {
                        const float4 x = load4(p.q, at + d);
                        top = max(max(top, __float_as_uint(x.x) & 0x7fffffffu), __float_as_uint(x.y) & 0x7fffffffu);
                        top = max(max(top, __float_as_uint(x.z) & 0x7fffffffu), __float_as_uint(x.w) & 0x7fffffffu);
                    }
                int e2 = static_cast<int>(top >> 23) - 127;
                e2 = top >= 0x7f800000u || top == 0 ? 0 : max(-120, min(120, e2));
                const float down = __uint_as_float(static_cast<uint32_t>(127 - e2) << 23);
                c *= __uint_as_float(static_cast<uint32_t>(127 + e2) << 23);
                uint8_t *dst = s_q + t * L::kQTile + row * 128;
#pragma unroll
                for (int d = 0; d < DP; d += 8) {
                    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f), y = x;
                    if (valid && d < p.dim) {
                        x = load4(p.q, at + d);
                        y = load4(p.q, at + d + 4);
                    }
                    *reinterpret_cast<uint4 *>(dst + (d >> 6) * L::kQHalf + ((((d & 63) >> 3) ^ (row & 7)) << 4)) =
                        make_uint4(pack16<false>(x.x * down, x.y * down), pack16<false>(x.z * down, x.w * down),
                                   pack16<false>(y.x * down, y.y * down), pack16<false>(y.z * down, y.w * down));
                }
                fence_proxy_async_smem();
                mbar_arrive(&bars.q_full);
            }
            float m = -INFINITY, l = 0.0f;  // m: the reference maximum of score * c (and log2 of sv's ratio), in base 2
            bool ok = true, nan = false;  // nan: the row sees a scale that is not finite
            for (int j = 0; j < n; j++) {
                const uint32_t s_at = s_cols + kTileKeys * (j % kBuffers);
                if (!mbar_wait_warp(&bars.s_full[t][j % kBuffers], (j / kBuffers) & 1, abort, status)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                uint32_t s[kTileKeys];
#pragma unroll
                for (int b = 0; b < kTileKeys; b += 32) tmem_ld32_start(s_at + b, s + b);
                tmem_ld_wait();
                const int k0 = range.token(j, kTileKeys);
                if (k0 + kTileKeys - 1 > t_lo || (p.window && k0 <= t_hi - p.window)) {
                    const int hi = pos - k0, lo = p.window ? hi - p.window + 1 : 0, sink = p.sinks - k0;
#pragma unroll
                    for (int b = 0; b < kTileKeys; b++)
                        if (b > hi || (b < lo && b >= sink)) s[b] = 0xff800000u;
                }
                float f[kTileKeys / 16];  // factor of the scores of 16 keys
                if (PAGED) {
                    if (!mbar_wait_warp(&bars.scales_full[j % kScaleSlots], (j / kScaleSlots) & 1, abort, status)) {
                        ok = false;
                        break;
                    }
#pragma unroll
                    for (int b = 0; b < kTileKeys / 16; b++) f[b] = c * bars.sk[j % kScaleSlots][b];
                    if (const uint32_t bad = bars.bad[j % kScaleSlots])
                        for (int b = 0; b < kTileKeys / 16; b++) {
                            const int key = k0 + 16 * b;
                            if (bad >> (8 * b) & 1) nan |= key <= pos && (!p.window || key + 15 > pos - p.window || key < p.sinks);
                        }
                }
                float mx = -INFINITY;
                if (PAGED) {
#pragma unroll
                    for (int b = 0; b < kTileKeys / 16; b++) {
                        float x = __uint_as_float(s[16 * b]), y = __uint_as_float(s[16 * b + 1]);
#pragma unroll
                        for (int e = 2; e < 14; e += 4) {
                            x = max3(x, __uint_as_float(s[16 * b + e]), __uint_as_float(s[16 * b + e + 1]));
                            y = max3(y, __uint_as_float(s[16 * b + e + 2]), __uint_as_float(s[16 * b + e + 3]));
                        }
                        x = max3(x, __uint_as_float(s[16 * b + 14]), __uint_as_float(s[16 * b + 15]));
                        mx = fmaxf(mx, fmaf(fmaxf(x, y), f[b], bars.lv[j % kScaleSlots][b]));
                    }
                } else {
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int b = 0; b < kTileKeys; b += 8)
#pragma unroll
                        for (int e = 0; e < 4; e++) top[e] = max3(top[e], __uint_as_float(s[b + e]), __uint_as_float(s[b + 4 + e]));
                    mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * c;
                }
                if (__any_sync(0xffffffffu, valid && mx - m > kLazy)) {  // (rows without a query hold what was there before)
                    const float to = fmaxf(m, mx);
                    const float keep = m == -INFINITY ? 0.0f : exp2f(m - to);
                    m = to;
                    l *= keep;
                    if (j > 0) {  // P.V(j - 1) of all tiles is in (P.V(j) waits for this row, so no later phase can be over)
                        if (!mbar_wait_warp(&bars.v_empty[(j - 1) % kStages], ((j - 1) / kStages) & 1, abort, status)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
#pragma unroll
                        for (int b = 0; b < DP; b += 32) {
                            uint32_t o[32];
                            tmem_ld32_start(o_at + b, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                            tmem_st32(o_at + b, o);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.0f : (PAGED || !BF16 ? kF16Up : 0.0f) - m;
                f32x2 sum[2] = {0, 0};
#pragma unroll
                for (int b = 0; b < kTileKeys / 32; b++) {
                    uint32_t w[16];
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        const int at = 32 * b + 16 * q;
                        const float fb = PAGED ? f[2 * b + q] : c, rb = PAGED ? ref + bars.lv[j % kScaleSlots][2 * b + q] : ref;
                        const f32x2 f2 = pair_of(fb, fb), r2 = pair_of(rb, rb);
                        f32x2 part[2] = {0, 0};
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const f32x2 x = fma2(pair_of(__uint_as_float(s[at + 2 * e]), __uint_as_float(s[at + 2 * e + 1])), f2, r2);
                            const float2 v = floats_of(x), a = make_float2(exp2_sfu(v.x), exp2_sfu(v.y));
                            f32x2 &to = PAGED ? part[e & 1] : sum[e & 1];
                            to = add2(to, pair_of(a.x, a.y));
                            w[8 * q + e] = pack16<BF16 && !PAGED>(a.x, a.y);
                        }
                        if (PAGED) {
                            const float iv = bars.iv[j % kScaleSlots][2 * b + q];
                            sum[q] = fma2(add2(part[0], part[1]), pair_of(iv, iv), sum[q]);
                        }
                    }
                    if (kTileKeys == 128 && b == 2) {  // P.V of the first half may begin
                        tmem_st_wait();
                        tc_fence_before();
                        mbar_arrive(&bars.p_full[t][0]);
                    }
                    tmem_st16_start(s_at + 16 * b, w);
                }
                const float2 s2 = floats_of(add2(sum[0], sum[1]));
                l += s2.x + s2.y;
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(&bars.p_full[t][kBuffers == 2 ? j & 1 : 1]);
            }
            // ---- out = O / l ----
            if (ok && n > 0) {
                ok = mbar_wait_warp(&bars.o_full[t], 0, abort, status);
                tc_fence_after();
            }
            if (ok) {
                const float inv = nan ? __uint_as_float(0x7fc00000u) : m == -INFINITY && l == 0.0f ? 0.0f : 1.0f / l;
                const float unit = PAGED && n > 0 ? bars.v_top : 1.0f;
                const long long at = (sq.q0 + i) * p.out.ts + (kvh * group + chunk * tl.heads + head) * p.out.hs;
                bool odd = false;  // something is not finite
#pragma unroll
                for (int b = 0; b < DP; b += 32) {
                    uint32_t o[32];
                    if (n > 0) {
                        tmem_ld32_start(o_at + b, o);
                        tmem_ld_wait();
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        uint32_t w[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            float v0 = n > 0 ? __uint_as_float(o[e + 2 * k]) * inv : 0.0f, v1 = n > 0 ? __uint_as_float(o[e + 2 * k + 1]) * inv : 0.0f;
                            if (PAGED) v0 *= unit, v1 *= unit;
                            odd |= !(fabsf(v0) <= 3.4e38f && fabsf(v1) <= 3.4e38f);
                            w[k] = pack16<BF16>(v0, v1);
                        }
                        if (valid && b + e < p.dim && p.out.vec)
                            *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.out.p) + at + b + e) = make_uint4(w[0], w[1], w[2], w[3]);
                        else if (valid && b + e < p.dim)
#pragma unroll
                            for (int k = 0; k < 8; k++) static_cast<uint16_t *>(p.out.p)[at + b + e + k] = static_cast<uint16_t>(w[k / 2] >> (16 * (k & 1)));
                    }
                }
                uint32_t again = __ballot_sync(0xffffffffu, valid && odd && !nan);
                while (again) {
                    const int from = __ffs(again) - 1;
                    again &= again - 1;
                    const int r_i = __shfl_sync(0xffffffffu, i, from), r_head = __shfl_sync(0xffffffffu, head, from);
                    compute_row<PAGED>(p, seq, sq.q0 + r_i, kvh * group + chunk * tl.heads + r_head, first + r_i, sq.k0, lane);
                }
            }
        }
    }
    // a wait that ran out: what this CTA has under way (loads, MMAs) gets 0.1 ms before its memory goes to another
    if (*abort)
        for (int i = 0; i < 100; i++) __nanosleep(1000);
    tc_fence_before();
    __syncthreads();
    if (warp == S::kIssuer) {
        tc_fence_after();
        tmem_dealloc(tmem, S::kTmem);
    }
}

bool rows_map(CUtensorMap *map, const Rows &r, int dim, int rows, int box_heads, int box_rows) {
    const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)r.heads, (cuuint64_t)rows};
    const cuuint64_t strides[2] = {(cuuint64_t)(r.heads == 1 ? dim * 2 : r.hs * 2), (cuuint64_t)r.ts * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows};
    return tensor_map(map, r.dtype == kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, r.p, dims,
                      strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

Tiling tiling_of(int group) {
    Tiling tl;
    tl.chunks = (group + kTileRows - 1) / kTileRows;
    tl.heads = (group + tl.chunks - 1) / tl.chunks;
    tl.toks = kTileRows / tl.heads;
    return tl;
}

template <int DP, bool BF16, bool FP8, class S>
cudaError_t launch(const TiledParams &p, cudaStream_t s) {
    const Tiling tl = tiling_of(p.q.heads / p.kv_heads);
    CUtensorMap q{}, k{}, v{};
    if (!S::kPaged && (!rows_map(&q, p.q, p.dim, p.n_q, tl.heads, tl.toks) ||
                       !rows_map(&k, p.rows.k, p.dim, p.rows.n_kv, 1, S::kKeys) || !rows_map(&v, p.rows.v, p.dim, p.rows.n_kv, 1, S::kKeys)))
        return cudaErrorInvalidValue;
    static SmemOptIn opt_in;
    const cudaError_t e = opt_in.set(reinterpret_cast<const void *>(k_tiled<DP, BF16, FP8, S>), Layout<DP, S>::kBytes);
    if (e != cudaSuccess) return e;
    const int pairs = (p.max_q + S::kTiles * tl.toks - 1) / (S::kTiles * tl.toks);
    const long long nx = (long long)pairs * p.kv_heads * tl.chunks;
    if (p.n_seqs > kTiledSeqs || nx > 0x7fffffffLL) return cudaErrorInvalidValue;
    k_tiled<DP, BF16, FP8, S><<<dim3((unsigned)nx, (unsigned)p.n_seqs), S::kThreads, Layout<DP, S>::kBytes, s>>>(q, k, v, p, tl, pairs);
    return cudaGetLastError();
}

// Keys in sight of a row from which the shape with the least MMA time wins.
constexpr long long kLongRun = 2048;

template <int DP, bool BF16>
cudaError_t launch_rows(const TiledParams &p, long long seen, cudaStream_t s) {
    if (seen >= kLongRun) return launch<DP, BF16, false, Shape<false, 128, 2>>(p, s);
    return launch<DP, BF16, false, Shape<false, 64, 1>>(p, s);
}

}  // namespace

cudaError_t window_attention(const WindowParams &w, int, cudaStream_t s) {
    TiledParams p{};
    p.q = w.q;
    p.out = w.out;
    p.qo = w.b.qo;
    p.n_seqs = w.b.n_seqs;
    p.n_q = w.b.n_q;
    p.max_q = w.b.max_q;
    p.kv_heads = w.k.heads;
    p.dim = w.dim;
    p.scale = w.scale;
    p.window = w.window;
    p.sinks = w.sinks;
    p.status = w.status;
    p.rows = Contiguous{w.k, w.v, w.b.ko, w.b.n_kv, w.b.max_kv};
    if (!p.q.vec || !w.k.vec || !w.v.vec || !p.out.vec || w.b.n_kv == 0) {
        const long long rows = (long long)p.n_q * p.q.heads;
        k_window_rows<<<(unsigned)((rows + kRowWarps - 1) / kRowWarps), kRowWarps * 32, 0, s>>>(p);
        return cudaGetLastError();
    }
    long long seen = w.b.max_kv;
    if (p.window) seen = std::min<long long>(seen, (long long)p.window + p.sinks);
    if (p.q.dtype == kBf16) return p.dim <= 64 ? launch_rows<64, true>(p, seen, s) : launch_rows<128, true>(p, seen, s);
    return p.dim <= 64 ? launch_rows<64, false>(p, seen, s) : launch_rows<128, false>(p, seen, s);
}

using CacheShape = Shape<true, 64, 2>;

// Rounds of CTAs, one to an SM, times tiles of keys.
double tiled_rounds(const AttendParams &a, int sms, long long seen) {
    const Tiling tl = tiling_of(a.q.heads / a.c.heads);
    const long long items = (long long)a.b.n_seqs * a.c.heads * tl.chunks * ((a.b.max_new + 2 * tl.toks - 1) / (2 * tl.toks));
    return (double)((items + sms - 1) / sms) * ((seen + CacheShape::kKeys - 1) / CacheShape::kKeys);
}

cudaError_t attend_tiled(const AttendParams &a, cudaStream_t s) {
    TiledParams p{};
    p.q = a.q;
    p.out = a.out;
    p.n_seqs = a.b.n_seqs;
    p.n_q = a.b.n_tokens;
    p.max_q = a.b.max_new;
    p.kv_heads = a.c.heads;
    p.dim = a.c.dim;
    p.scale = a.scale;
    p.window = a.window;
    p.sinks = a.sinks;
    p.status = a.status;
    p.paged = Paged{a.c, a.b};
    const bool bf16 = a.out.dtype == kBf16;
    if (p.dim <= 64) {
        if (a.c.fp8) return bf16 ? launch<64, true, true, CacheShape>(p, s) : launch<64, false, true, CacheShape>(p, s);
        return bf16 ? launch<64, true, false, CacheShape>(p, s) : launch<64, false, false, CacheShape>(p, s);
    }
    if (a.c.fp8) return bf16 ? launch<128, true, true, CacheShape>(p, s) : launch<128, false, true, CacheShape>(p, s);
    return bf16 ? launch<128, true, false, CacheShape>(p, s) : launch<128, false, false, CacheShape>(p, s);
}

}  // namespace kv
}  // namespace ditch
