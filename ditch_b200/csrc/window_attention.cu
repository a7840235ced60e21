// Causal attention with a sliding window and sinks over contiguous f16 / bf16
// rows, on the fifth-generation tensor cores.
//
// Bound by the tensor cores and, just as much, by the exponentials: a 128 x
// 128 tile of scores takes 512 cycles of MMA for Q.K^T, 512 for P.V (head
// size 128) and 1024 cycles of the SFU. One CTA therefore works on two tiles
// of 128 query rows, whose products and softmax alternate:
//   warps 0-3, 4-7   softmax of the first and second row tile, a row a thread
//   warp 8           issues the MMAs (one thread)
//   warp 9           loads (one thread)
// A row tile is all the query heads of one key / value head for as many
// tokens as fill 128 rows, so both tiles read the same keys and values, and a
// window or the causal limit cuts as close as a few tokens.
//
// TMEM: S of both tiles (128 columns each), O of both (128 each). P goes back
// over its S as 16-bit pairs and is the A operand of P.V from there; V is
// taken as it lies, [token][dimension], as a transposed (MN-major) B operand.
// The MMAs of one CTA complete in the order of their issue, so S(j + 1) of a
// tile may be issued right behind P.V(j), and when S(j + 1) is there, O has
// taken in P(j): a row whose maximum has grown by more than 2^kLazy since its
// sums' reference rescales its part of O in TMEM then; most never do.
//
// What a row does not see has weight 0 in the product, and 0 times an
// infinity or NaN is NaN: rows whose result is not finite are computed again
// from the keys that they do see (recompute_row).
//
// Rows that TMA cannot take (not 16-byte aligned) go by k_window_rows, one
// warp for each row.
#include <algorithm>

#include "attn_common.cuh"
#include "gemm.cuh"
#include "kv_range.cuh"

namespace ditch {
namespace kv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.0f;  // a weight stays below 2^8
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
        const float top = fmaxf(m, s);
        const float keep = top == -INFINITY ? 1.0f : exp2f(m - top), w = top == -INFINITY ? 0.0f : exp2f(s - top);
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

// Query row `tok` of head `head`, at position pos of the sequence whose keys
// begin at row k0.
__device__ __noinline__ void compute_row(const WindowParams &p, int tok, int head, int pos, int k0, int lane) {
    const int d = 4 * lane, kvh = head / (p.q.heads / p.k.heads);
    float q[4] = {0, 0, 0, 0};
    for (int e = 0; e < 4; e++)
        if (d + e < p.dim) q[e] = load1(p.q, tok * p.q.ts + head * p.q.hs + d + e);
    RowState st;
    for (int j = first_key(pos, p.window, p.sinks); j <= pos; j = next_key(j, pos, p.window, p.sinks)) {
        float k[4] = {0, 0, 0, 0}, v[4] = {0, 0, 0, 0};
        for (int e = 0; e < 4; e++)
            if (d + e < p.dim) {
                k[e] = load1(p.k, (k0 + j) * p.k.ts + kvh * p.k.hs + d + e);
                v[e] = load1(p.v, (k0 + j) * p.v.ts + kvh * p.v.hs + d + e);
            }
        st.key(q, k, v, p.scale * kLog2e);
    }
    for (int e = 0; e < 4; e++)
        if (d + e < p.dim) store1(p.out, tok * p.out.ts + head * p.out.hs + d + e, st.m == -INFINITY && st.sum == 0.0f ? 0.0f : st.o[e] / st.sum);
}

// Sequence `seq` of the batch: its query and key rows, none (and the status
// word set) when the device's numbers leave the host's bounds.
struct Seq {
    int q0, nq, k0, nk;
};

__device__ __forceinline__ Seq seq_of(const Ragged &b, int seq, int *status) {
    Seq s;
    s.q0 = __ldg(b.qo + seq);
    s.k0 = __ldg(b.ko + seq);
    const int q1 = __ldg(b.qo + seq + 1), k1 = __ldg(b.ko + seq + 1);
    s.nq = q1 - s.q0;
    s.nk = k1 - s.k0;
    if (s.q0 < 0 || q1 > b.n_q || s.nq < 0 || s.nq > b.max_q || s.k0 < 0 || k1 > b.n_kv || s.nk < 0 || s.nk > b.max_kv) {
        flag(status);
        s.nq = s.nk = 0;
    }
    return s;
}

__global__ void __launch_bounds__(kRowWarps * 32) k_window_rows(WindowParams p) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long row = static_cast<long long>(blockIdx.x) * kRowWarps + warp;
    if (row >= static_cast<long long>(p.b.n_q) * p.q.heads) return;
    const int tok = static_cast<int>(row / p.q.heads), head = static_cast<int>(row % p.q.heads);
    int seq = 0;
    while (seq + 1 < p.b.n_seqs && __ldg(p.b.qo + seq + 1) <= tok) seq++;
    const Seq s = seq_of(p.b, seq, p.status);
    if (tok < s.q0 || tok >= s.q0 + s.nq) return;
    compute_row(p, tok, head, s.nk - s.nq + tok - s.q0, s.k0, lane);
}

// ---- the tiled kernel ------------------------------------------------------------------
constexpr int kTileRows = 128;  // query rows of a tile: the MMA's M, a TMEM lane each
constexpr int kTileKeys = 128;
constexpr int kBoxKeys = 64;    // keys of one TMA box
constexpr int kStages = 2;
constexpr int kThreads = 320;

template <int DP>
struct WinLayout {
    static constexpr int kHalf = kTileRows * 128;             // 64 dimensions of 128 rows
    static constexpr int kTile = kHalf * (DP / 64);           // a tile of Q, K or V
    static constexpr int kBytes = 1024 + (2 + 2 * kStages) * kTile;
};

struct WinBars {
    uint64_t q_full, k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
    uint64_t s_full[2], p_full[2], o_full[2];
    uint32_t tmem;
    int abort;
};

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

__device__ __forceinline__ void tmem_ld32_ready(uint32_t *r) {
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]));
    asm volatile("" : "+r"(r[30]), "+r"(r[31]));
}

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

__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float exp2_sfu(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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

template <int DP, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    k_window(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
             const __grid_constant__ CUtensorMap v_map, WindowParams p, Tiling tl, int pairs) {
    using L = WinLayout<DP>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ WinBars bars;
    // the longest runs of keys first
    const int pair = pairs - 1 - blockIdx.y;
    int x = blockIdx.x;
    const int chunk = x % tl.chunks;
    x /= tl.chunks;
    const int kvh = x % p.k.heads, seq = x / p.k.heads;
    const Seq sq = seq_of(p.b, seq, p.status);
    const int i0 = pair * 2 * tl.toks;  // first token of the pair
    if (i0 >= sq.nq) return;
    const int tiles = i0 + tl.toks < sq.nq ? 2 : 1;
    const int group = p.q.heads / p.k.heads;
    const int first = sq.nk - sq.nq;  // position of the sequence's first query
    const int p_lo = first + i0, p_hi = first + min(sq.nq, i0 + 2 * tl.toks) - 1;
    Range range = range_of(max(p_lo, 0), max(p_hi, 0), p.window, p.sinks, kTileKeys);
    const int n = p_hi < 0 ? 0 : range.n;
    auto keys_of = [&](int j) {  // of tile j: up to the last row's position, in whole MMA steps
        return min(kTileKeys, (p_hi + 1 - range.token(j, kTileKeys) + 15) & ~15);
    };

    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *s_q = base, *s_k = base + 2 * L::kTile, *s_v = s_k + kStages * L::kTile;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        mbar_init(&bars.q_full, 1);
        for (int i = 0; i < kStages; i++) {
            mbar_init(&bars.k_full[i], 1);
            mbar_init(&bars.k_empty[i], 1);
            mbar_init(&bars.v_full[i], 1);
            mbar_init(&bars.v_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&bars.s_full[i], 1);
            mbar_init(&bars.p_full[i], kTileRows);
            mbar_init(&bars.o_full[i], 1);
        }
        bars.abort = 0;
        fence_barrier_init();
    }
    if (warp == 8) {
        tmem_alloc(&bars.tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars.tmem;
    int *status = p.status;
    volatile int *abort = &bars.abort;

    if (warp == 9) {
        if (lane == 0 && n > 0) {
            const int head0 = kvh * group + chunk * tl.heads;
            mbar_arrive_expect_tx(&bars.q_full, tiles * (DP / 64) * tl.heads * tl.toks * 128);
            for (int t = 0; t < tiles; t++)
#pragma unroll
                for (int h = 0; h < DP / 64; h++)
                    tma_load_rows(&q_map, &bars.q_full, s_q + t * L::kTile + h * L::kHalf, 64 * h, head0, sq.q0 + i0 + t * tl.toks);
            for (int j = 0; j < n; j++) {
                const int st = j % kStages, at = sq.k0 + range.token(j, kTileKeys);
                const int boxes = (keys_of(j) + kBoxKeys - 1) / kBoxKeys;
                for (int kv = 0; kv < 2; kv++) {
                    uint64_t *full = kv ? &bars.v_full[st] : &bars.k_full[st], *empty = kv ? &bars.v_empty[st] : &bars.k_empty[st];
                    if (j >= kStages && !mbar_wait(empty, (j / kStages + 1) & 1, abort, status)) goto loads_done;
                    mbar_arrive_expect_tx(full, boxes * (DP / 64) * kBoxKeys * 128);
                    uint8_t *dst = (kv ? s_v : s_k) + st * L::kTile;
                    for (int b = 0; b < boxes; b++)
#pragma unroll
                        for (int h = 0; h < DP / 64; h++)
                            tma_load_rows(kv ? &v_map : &k_map, full, dst + h * L::kHalf + b * kBoxKeys * 128, 64 * h, kvh,
                                          at + b * kBoxKeys);
                }
            }
        loads_done:;
        }
    } else if (warp == 8) {
        if (lane == 0 && n > 0) {
            constexpr uint32_t kType = BF16 ? 1 : 0;
            auto qk = [&](int t, int j) {
                const int st = j % kStages;
                const uint32_t id = idesc_of(kType, false, keys_of(j));
#pragma unroll
                for (int h = 0; h < DP / 64; h++) {
                    const uint64_t a = sw128_kmajor_desc(smem_u32(s_q + t * L::kTile + h * L::kHalf));
                    const uint64_t b = sw128_kmajor_desc(smem_u32(s_k + st * L::kTile + h * L::kHalf));
#pragma unroll
                    for (int k = 0; k < 4; k++) tc_mma_bf16(tmem + 128 * t, a + 2 * k, b + 2 * k, id, (h | k) ? 1u : 0u);
                }
                tc_commit(&bars.s_full[t]);
            };
            bool ok = mbar_wait(&bars.q_full, 0, abort, status) && mbar_wait(&bars.k_full[0], 0, abort, status);
            if (ok) {
                tc_fence_after();
                for (int t = 0; t < tiles; t++) qk(t, 0);
                tc_commit(&bars.k_empty[0]);
            }
            for (int j = 0; ok && j < n; j++) {
                const int st = j % kStages, steps = keys_of(j) / 16;
                for (int t = 0; ok && t < tiles; t++) {
                    ok = mbar_wait(&bars.p_full[t], j & 1, abort, status);
                    if (ok && t == 0) ok = mbar_wait(&bars.v_full[st], (j / kStages) & 1, abort, status);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t id = idesc_of(kType, true, DP);
                    const uint64_t v = sw128_mnmajor_desc(smem_u32(s_v + st * L::kTile), L::kHalf);
                    for (int k = 0; k < steps; k++)
                        tc_mma_ts(tmem + 256 + 128 * t, tmem + 128 * t + 8 * k, v + (k * 16 * 128 >> 4), id, (j | k) ? 1u : 0u);
                    if (t == tiles - 1) tc_commit(&bars.v_empty[st]);
                    if (j + 1 < n) {
                        if (t == 0) {
                            ok = mbar_wait(&bars.k_full[(j + 1) % kStages], ((j + 1) / kStages) & 1, abort, status);
                            if (!ok) break;
                            tc_fence_after();
                        }
                        qk(t, j + 1);
                        if (t == tiles - 1) tc_commit(&bars.k_empty[(j + 1) % kStages]);
                    } else {
                        tc_commit(&bars.o_full[t]);
                    }
                }
            }
        }
    } else if ((warp >> 2) < tiles) {
        // ---- softmax of tile t: this thread's row ----
        const int t = warp >> 2, row = tid & 127;
        const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
        const uint32_t s_at = tmem + lanes + 128 * t, o_at = tmem + lanes + 256 + 128 * t;
        const int tok = row / tl.heads, head = row - tok * tl.heads;  // of the tile
        const int i = i0 + t * tl.toks + tok, pos = first + i;
        const bool valid = tok < tl.toks && i < sq.nq && chunk * tl.heads + head < group;
        // the tile's rows: the tiles of keys that all of them see whole need no masks
        const int t_lo = first + i0 + t * tl.toks, t_hi = min(t_lo + tl.toks, first + sq.nq) - 1;
        const float c = p.scale * kLog2e;
        float m = -INFINITY, l = 0.0f;  // m in units of the scores
        bool ok = true;
        for (int j = 0; j < n; j++) {
            if (!mbar_wait(&bars.s_full[t], j & 1, abort, status)) {
                ok = false;
                break;
            }
            tc_fence_after();
            uint32_t s[128];
#pragma unroll
            for (int b = 0; b < 4; b++) tmem_ld32_start(s_at + 32 * b, s + 32 * b);
            tmem_ld_wait();
#pragma unroll
            for (int b = 0; b < 4; b++) tmem_ld32_ready(s + 32 * b);
            const int k0 = range.token(j, kTileKeys);
            if (k0 + kTileKeys - 1 > t_lo || (p.window && k0 <= t_hi - p.window)) {
                const int hi = pos - k0, lo = p.window ? hi - p.window + 1 : 0, sink = p.sinks - k0;
#pragma unroll
                for (int b = 0; b < 128; b++)
                    if (b > hi || (b < lo && b >= sink)) s[b] = 0xff800000u;
            }
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int b = 0; b < 128; b += 8)
#pragma unroll
                for (int e = 0; e < 4; e++) top[e] = fmaxf(top[e], fmaxf(__uint_as_float(s[b + e]), __uint_as_float(s[b + 4 + e])));
            const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            if (__any_sync(0xffffffffu, (mx - m) * c > kLazy)) {
                const float to = fmaxf(m, mx);
                const float keep = m == -INFINITY ? 0.0f : exp2f((m - to) * c);
                m = to;
                l *= keep;
                if (j > 0) {
#pragma unroll
                    for (int b = 0; b < DP; b += 32) {
                        uint32_t o[32];
                        tmem_ld32_start(o_at + b, o);
                        tmem_ld_wait();
                        tmem_ld32_ready(o);
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                        tmem_st32(o_at + b, o);
                    }
                }
            }
            const float ref = m == -INFINITY ? 0.0f : -m * c;
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int b = 0; b < 2; b++) {
                uint32_t w[32];
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    const float a0 = exp2_sfu(fmaf(__uint_as_float(s[64 * b + 2 * e]), c, ref));
                    const float a1 = exp2_sfu(fmaf(__uint_as_float(s[64 * b + 2 * e + 1]), c, ref));
                    sum[(2 * e) & 3] += a0;
                    sum[(2 * e + 1) & 3] += a1;
                    w[e] = pack16<BF16>(a0, a1);
                }
                tmem_st32(s_at + 32 * b, w);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(&bars.p_full[t]);
        }
        // ---- out = O / l ----
        if (ok && n > 0) {
            ok = mbar_wait(&bars.o_full[t], 0, abort, status);
            tc_fence_after();
        }
        if (ok) {
            const float inv = m == -INFINITY && l == 0.0f ? 0.0f : 1.0f / l;
            const long long at = (sq.q0 + i) * p.out.ts + (kvh * group + chunk * tl.heads + head) * p.out.hs;
            bool odd = false;  // something is not finite
#pragma unroll
            for (int b = 0; b < DP; b += 32) {
                uint32_t o[32];
                if (n > 0) {
                    tmem_ld32_start(o_at + b, o);
                    tmem_ld_wait();
                    tmem_ld32_ready(o);
                }
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const float v0 = n > 0 ? __uint_as_float(o[e + 2 * k]) * inv : 0.0f, v1 = n > 0 ? __uint_as_float(o[e + 2 * k + 1]) * inv : 0.0f;
                        odd |= !(fabsf(v0) <= 3.4e38f && fabsf(v1) <= 3.4e38f);
                        w[k] = pack16<BF16>(v0, v1);
                    }
                    if (valid && b + e < p.dim)
                        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.out.p) + at + b + e) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            uint32_t again = __ballot_sync(0xffffffffu, valid && odd);
            while (again) {
                const int from = __ffs(again) - 1;
                again &= again - 1;
                const int r_i = __shfl_sync(0xffffffffu, i, from), r_head = __shfl_sync(0xffffffffu, head, from);
                compute_row(p, sq.q0 + r_i, kvh * group + chunk * tl.heads + r_head, first + r_i, sq.k0, lane);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

bool rows_map(CUtensorMap *map, const Rows &r, int dim, int rows, int box_heads, int box_rows) {
    const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)r.heads, (cuuint64_t)rows};
    const cuuint64_t strides[2] = {(cuuint64_t)(r.heads == 1 ? dim * 2 : r.hs * 2), (cuuint64_t)r.ts * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows};
    return tensor_map(map, r.dtype == kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, r.p, dims,
                      strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int DP, bool BF16>
cudaError_t launch(const WindowParams &p, cudaStream_t s) {
    const int group = p.q.heads / p.k.heads;
    Tiling tl;
    tl.chunks = (group + kTileRows - 1) / kTileRows;
    tl.heads = (group + tl.chunks - 1) / tl.chunks;
    tl.toks = kTileRows / tl.heads;
    CUtensorMap q, k, v;
    if (!rows_map(&q, p.q, p.dim, p.b.n_q, tl.heads, tl.toks) || !rows_map(&k, p.k, p.dim, p.b.n_kv, 1, kBoxKeys) ||
        !rows_map(&v, p.v, p.dim, p.b.n_kv, 1, kBoxKeys))
        return cudaErrorInvalidValue;
    static SmemOptIn opt_in;
    const cudaError_t e = opt_in.set(reinterpret_cast<const void *>(k_window<DP, BF16>), WinLayout<DP>::kBytes);
    if (e != cudaSuccess) return e;
    const int pairs = (p.b.max_q + 2 * tl.toks - 1) / (2 * tl.toks);
    const long long nx = (long long)p.b.n_seqs * p.k.heads * tl.chunks;
    if (pairs > 65535 || nx > 0x7fffffffLL) return cudaErrorInvalidValue;
    k_window<DP, BF16><<<dim3((unsigned)nx, (unsigned)pairs), kThreads, WinLayout<DP>::kBytes, s>>>(q, k, v, p, tl, pairs);
    return cudaGetLastError();
}

}  // namespace

cudaError_t window_attention(const WindowParams &p, int, cudaStream_t s) {
    if (!p.q.vec || !p.k.vec || !p.v.vec || !p.out.vec || p.b.n_kv == 0) {
        const long long rows = (long long)p.b.n_q * p.q.heads;
        k_window_rows<<<(unsigned)((rows + kRowWarps - 1) / kRowWarps), kRowWarps * 32, 0, s>>>(p);
        return cudaGetLastError();
    }
    if (p.q.dtype == kBf16) return p.dim <= 64 ? launch<64, true>(p, s) : launch<128, true>(p, s);
    return p.dim <= 64 ? launch<64, false>(p, s) : launch<128, false>(p, s);
}

}  // namespace kv
}  // namespace ditch
