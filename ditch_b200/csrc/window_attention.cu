// Attention over contiguous rows: one warp per (row, query head), keys one by one with a running maximum and sum.
#include "attn_common.cuh"
#include "kvcache.cuh"

namespace ditch {
namespace kv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRowWarps = 4;

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

__global__ void __launch_bounds__(kRowWarps * 32) k_window_rows(WindowParams p) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = 4 * lane;
    const long long row = static_cast<long long>(blockIdx.x) * kRowWarps + warp;
    if (row >= static_cast<long long>(p.b.n_q) * p.q.heads) return;
    const int tok = static_cast<int>(row / p.q.heads), head = static_cast<int>(row % p.q.heads);
    int seq = 0;
    while (seq + 1 < p.b.n_seqs && __ldg(p.b.qo + seq + 1) <= tok) seq++;
    const int q0 = p.b.qo[seq], q1 = p.b.qo[seq + 1], k0 = p.b.ko[seq], k1 = p.b.ko[seq + 1];
    if (q0 < 0 || q1 > p.b.n_q || tok < q0 || tok >= q1 || k0 < 0 || k1 > p.b.n_kv || k1 < k0) {
        flag(p.status);
        return;
    }
    const int pos = (k1 - k0) - (q1 - q0) + (tok - q0), kvh = head / (p.q.heads / p.k.heads);
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
        if (d + e < p.dim)
            store1(p.out, tok * p.out.ts + head * p.out.hs + d + e, st.m == -INFINITY ? 0.0f : st.o[e] / st.sum);
}

}  // namespace

cudaError_t window_attention(const WindowParams &p, int, cudaStream_t s) {
    const long long rows = (long long)p.b.n_q * p.q.heads;
    k_window_rows<<<(unsigned)((rows + kRowWarps - 1) / kRowWarps), kRowWarps * 32, 0, s>>>(p);
    return cudaGetLastError();
}

}  // namespace kv
}  // namespace ditch
