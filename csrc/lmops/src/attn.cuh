// attn.cuh — what the window-attention kernels share: the mask and the list
// of key tiles of a query tile (and of query tiles of a key tile).
#pragma once
#include "ops_common.cuh"

namespace cailops {

struct AttnArgs {
    int B, T, H, Hkv, D, group;
    int window, sinks;
    float scale, scale_log2;  // scale, scale * log2(e)
    const int32_t *lengths;
    const char *q, *k, *v, *dout;
    char *o, *rest, *dq, *dk, *dv;
    // strides in bytes
    int64_t qb, qt, qh, kb, kt, kh, vb, vt, vh, ob, ot, oh;
    int64_t rb, rt, rh;  // rest
    int rest_rows;       // the first rows of a sequence, whose rest is kept
    int fine_rows;       // and whose p is rounded to twice the bits
    int64_t gb, gt, gh;  // dout
    int64_t dqb, dqt, dqh, dkb, dkt, dkh, dvb, dvt, dvh;
    float *lse, *delta;  // [B, H] rows of `lse_row` values; lse in log2 units of the scaled scores
    int64_t lse_row;     // T rounded up to 4
    int *error;          // the device's error word (kernels with bounded waits)
};

// fills everything but D-dependent launch choices; 0 or an error code
int attn_check(const cail_ops_attention_args *a, bool backward, const char *who);
AttnArgs attn_args(const cail_ops_attention_args *a, bool backward);

// The sinks' key tiles are seen by all queries; in backward their queries are
// cut into parts where they would be the last blocks running, and the parts'
// sums joined in order.
struct SinkParts {
    int splits, tiles;  // parts of a key tile, key tiles with sinks (1 and 0: none is cut)
    float *sums;        // [B, Hkv, tiles, splits, 2, rows of a tile, DP]: partial dk and dv
};
// for blocks of `rows` keys that go over tiles of `stream` queries, `slots` of them at a time
SinkParts sink_parts(const cail_ops_attention_args *a, int rows, int stream, int64_t slots);
inline size_t sink_bytes(const cail_ops_attention_args *a, const SinkParts &p, int rows, int dp) {
    return p.splits > 1 ? (size_t)a->B * a->Hkv * p.tiles * p.splits * 2 * rows * dp * sizeof(float) : 0;
}

// The tensor-core kernels' grids: heads, sequences, then tiles of 128 rows, so
// that blocks start in the tiles' order and find their place without a division.
constexpr int kMostTiles = 65535;

// the tensor-core path (attn_tc_*.cu): whether it takes the call, and the call
bool tc_takes(const cail_ops_attention_args *a);
bool tc_takes_backward(const cail_ops_attention_args *a);
bool tc_takes_decode(const cail_ops_attention_args *a);
int tc_decode(const cail_ops_attention_args *a, cudaStream_t st);
int tc_forward(const cail_ops_attention_args *a, cudaStream_t st);
int tc_backward(const cail_ops_attention_args *a, cudaStream_t st);
size_t tc_workspace(const cail_ops_attention_args *a);

#ifdef __CUDACC__
// dk and dv of the sinks' key tiles from their parts, in order
template <typename T, int DP, int ROWS> __global__ void __launch_bounds__(256) join_kernel(const AttnArgs a, const SinkParts parts) {
    const int hk = blockIdx.y, b = blockIdx.z;
    const int64_t tile0 = ((int64_t)b * a.Hkv + hk) * parts.tiles;
    for (int i = blockIdx.x * 256 + threadIdx.x; i < parts.tiles * 2 * ROWS * (DP / 4); i += gridDim.x * 256) {
        const int d = (i % (DP / 4)) * 4, row = i / (DP / 4) % ROWS, which = i / (DP / 4) / ROWS % 2, tile = i / (DP / 4) / ROWS / 2;
        const int j = tile * ROWS + row;
        if (j >= a.T || d >= a.D) continue;
        float s[4] = {};
        for (int p = 0; p < parts.splits; ++p) {
            const float4 x = *reinterpret_cast<const float4 *>(parts.sums + ((((tile0 + tile) * parts.splits + p) * 2 + which) * ROWS + row) * DP + d);
            s[0] += x.x, s[1] += x.y, s[2] += x.z, s[3] += x.w;
        }
        T *out = reinterpret_cast<T *>(which ? a.dv + b * a.dvb + (int64_t)j * a.dvt + hk * a.dvh : a.dk + b * a.dkb + (int64_t)j * a.dkt + hk * a.dkh);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < a.D) out[d + e] = from_f<T>(s[e]);
    }
}
template <typename T, int DP, int ROWS> int join(const AttnArgs &a, const SinkParts &parts, cudaStream_t st) {
    const unsigned grid = ((unsigned)parts.tiles * 2 * ROWS * (DP / 4) + 255) / 256;
    join_kernel<T, DP, ROWS><<<dim3(grid < 1024u ? grid : 1024u, a.Hkv, a.B), 256, 0, st>>>(a, parts);
    return launched("window attention backward");
}

__device__ __forceinline__ bool seen(int i, int j, int n, int window, int sinks) {
    return i < n && j <= i && (i - j < window || j < sinks);
}

// what rounding to T takes from x
template <typename T> __device__ __forceinline__ float rest_of(float x) { return x - to_f(from_f<T>(x)); }

// A row that sees one key: its probability is 1 whatever the scores, so no
// gradient reaches q and k through it.  (p (dp - delta) would leave the
// difference of two roundings where the result is zero.)
__device__ __forceinline__ bool one_key(int i, int window, int sinks) { return i == 0 || (window == 1 && sinks == 0); }

// The key tiles (of TK keys) that the query rows [i0, i1) of a sequence of n
// tokens need, in order: [0, sink_end) and [win_begin, win_end).
struct KeyTiles {
    int sink_end, win_begin, count;
    __device__ __forceinline__ KeyTiles(int i0, int i1, int n, int window, int sinks, int tile) {
        i1 = min(i1, n);
        if (i0 >= i1) {
            sink_end = win_begin = count = 0;
            return;
        }
        const int win_end = (i1 - 1) / tile + 1;
        win_begin = window > i0 ? 0 : (i0 - window + 1) / tile;
        sink_end = sinks > 0 ? min((min(sinks, n) - 1) / tile + 1, win_begin) : 0;
        count = sink_end + win_end - win_begin;
    }
    __device__ __forceinline__ int at(int x) const { return x < sink_end ? x : x - sink_end + win_begin; }
};

// The query rows that see some key of [j0, j1): [begin, end)
__device__ __forceinline__ void query_range(int j0, int j1, int n, int window, int sinks, int &begin, int &end) {
    begin = j0;
    const int64_t last = (int64_t)min(j1, n) - 1 + window;  // the last row the window reaches, plus one
    end = j0 < sinks ? n : (int)min((int64_t)n, last);
    if (j0 >= n) begin = end = 0;
}

// bits [lo, hi] of 32 (none where lo > hi); lo and hi may lie outside
__device__ __forceinline__ uint32_t bits(int lo, int hi) {
    if (lo > hi || lo > 31 || hi < 0) return 0u;
    return (0xffffffffu << max(lo, 0)) & (0xffffffffu >> (31 - min(hi, 31)));
}
// which of the keys j0 .. j0 + 31 row i sees (i < n)
__device__ __forceinline__ uint32_t keys_of_row(int i, int j0, int window, int sinks) {
    return bits(i - window + 1 - j0, i - j0) | bits(0, min(sinks - 1, i) - j0);
}
// which of the rows i0 .. i0 + 31 see key j
__device__ __forceinline__ uint32_t rows_of_key(int j, int i0, int n, int window, int sinks) {
    return bits(j - i0, (j < sinks || window > n - j ? n - 1 : j + window - 1) - i0) & bits(0, n - 1 - i0);
}

__device__ __forceinline__ int length_of(const AttnArgs &a, int b) {
    return a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
}
#endif

}  // namespace cailops
