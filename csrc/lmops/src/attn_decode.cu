// attn_decode.cu — one token per sequence against a cache.
//
// The keys that the token sees (the window and the sinks before it) are
// split over the blocks of a cluster, so one sequence and few heads still
// use many SMs; each block serves the query heads that share a key head, so
// the cache is read once per group.  A key row is held by a group of lanes
// (16 bytes each); every lane group keeps its own running maximum, sum and
// output for its keys, and the groups, warps and blocks join at the end:
// lanes by shuffles, warps through shared memory, blocks through distributed
// shared memory.  One launch, no workspace.  Bound by latency where it is used
// (1 sequence, 16 heads of 64, 256 keys: 5.3 us, of which 2.5 are the launch).
#include <cooperative_groups.h>

#include "attn.cuh"

namespace cg = cooperative_groups;

namespace cailops {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;

// E elements of a row at element c0; columns >= D as zeros
template <typename T, int E, bool VEC> __device__ __forceinline__ void load_row(const char *row, int c0, int D, float *x) {
    if constexpr (VEC) {
        Vec<T, E> v;
        if (c0 < D) v = *reinterpret_cast<const Vec<T, E> *>(row + c0 * sizeof(T));
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = c0 < D ? to_f(v.v[e]) : 0.f;
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = c0 + e < D ? to_f(reinterpret_cast<const T *>(row)[c0 + e]) : 0.f;
    }
}

// LANES hold a row of up to LANES * E elements; G query heads per block
template <typename T, int LANES, int G, bool VEC>
__global__ void __launch_bounds__(kThreads) decode_kernel(const AttnArgs a) {
    constexpr int E = 16 / (int)sizeof(T), DP = LANES * E, ROWS = 32 / LANES, U = G >= 4 ? 2 : 4;
    __shared__ float so[kWarps][G][DP];
    __shared__ float sm[kWarps][G], sl[kWarps][G];
    __shared__ float bo[G][DP], bm[G], bl[G];
    cg::cluster_group cl = cg::this_cluster();
    const int blocks = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int chunks = (a.group + G - 1) / G;
    const int b = blockIdx.z, hk = blockIdx.y / chunks, h0 = hk * a.group + (blockIdx.y % chunks) * G;
    const int heads = min(G, (hk + 1) * a.group - h0);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = lane / LANES, c0 = (lane % LANES) * E;
    const int n = length_of(a, b);

    // the keys it sees, numbered: the sinks before the window, then the window
    const int win0 = max(0, n - a.window), nsink = min(a.sinks, win0), keys = nsink + n - win0;
    const int per = (keys + blocks - 1) / blocks;
    const int from = min(keys, rank * per), to = min(keys, from + per);

    float q[G][E], o[G][E] = {}, m[G], l[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        m[g] = -INFINITY, l[g] = 0.f;
        if (g < heads) {
            load_row<T, E, VEC>(a.q + b * a.qb + (h0 + g) * a.qh, c0, a.D, q[g]);
#pragma unroll
            for (int e = 0; e < E; ++e) q[g][e] *= a.scale_log2;
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) q[g][e] = 0.f;
        }
    }
    const char *kp = a.k + b * a.kb + hk * a.kh, *vp = a.v + b * a.vb + hk * a.vh;
    for (int x0 = from + (warp * ROWS + sub); x0 - sub < to; x0 += kWarps * ROWS * U) {
        float k[U][E], v[U][E];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int x = x0 + u * kWarps * ROWS;
            const int64_t j = x < nsink ? x : x - nsink + win0;
            if (x < to) {
                load_row<T, E, VEC>(kp + j * a.kt, c0, a.D, k[u]);
                load_row<T, E, VEC>(vp + j * a.vt, c0, a.D, v[u]);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) k[u][e] = 0.f, v[u][e] = 0.f;
            }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float s[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s[u] = 0.f;
#pragma unroll
                for (int e = 0; e < E; ++e) s[u] = fmaf(q[g][e], k[u][e], s[u]);
            }
#pragma unroll
            for (int w = LANES / 2; w; w >>= 1)
#pragma unroll
                for (int u = 0; u < U; ++u) s[u] += __shfl_xor_sync(0xffffffffu, s[u], w);
            float top = m[g];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (x0 + u * kWarps * ROWS >= to) s[u] = -INFINITY;
                top = fmaxf(top, s[u]);
            }
            const float base = top == -INFINITY ? 0.f : top, turn = exp2_fast(m[g] - base);
            m[g] = top;
            l[g] *= turn;
#pragma unroll
            for (int e = 0; e < E; ++e) o[g][e] *= turn;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float p = exp2_fast(s[u] - base);
                l[g] += p;
#pragma unroll
                for (int e = 0; e < E; ++e) o[g][e] = fmaf(p, v[u][e], o[g][e]);
            }
        }
    }

    // lane groups of a warp
#pragma unroll
    for (int g = 0; g < G; ++g) {
        float top = m[g];
#pragma unroll
        for (int w = LANES; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        const float turn = exp2_fast(m[g] - (top == -INFINITY ? 0.f : top));
        l[g] *= turn;
#pragma unroll
        for (int e = 0; e < E; ++e) o[g][e] *= turn;
#pragma unroll
        for (int w = LANES; w < 32; w <<= 1) {
            l[g] += __shfl_xor_sync(0xffffffffu, l[g], w);
#pragma unroll
            for (int e = 0; e < E; ++e) o[g][e] += __shfl_xor_sync(0xffffffffu, o[g][e], w);
        }
        if (sub == 0) {
#pragma unroll
            for (int e = 0; e < E; ++e) so[warp][g][c0 + e] = o[g][e];
            if (lane == 0) sm[warp][g] = top, sl[warp][g] = l[g];
        }
    }
    __syncthreads();
    // warps of the block
    for (int i = tid; i < G * DP; i += kThreads) {
        const int g = i / DP, d = i % DP;
        float top = sm[0][g];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sm[w][g]);
        const float base = top == -INFINITY ? 0.f : top;
        float x = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = exp2_fast(sm[w][g] - base);
            x = fmaf(so[w][g][d], f, x);
            sum = fmaf(sl[w][g], f, sum);
        }
        bo[g][d] = x;
        if (d == 0) bm[g] = top, bl[g] = sum;
    }
    cl.sync();
    // blocks of the cluster: each joins a part of the output
    for (int i = rank * kThreads + tid; i < heads * a.D; i += blocks * kThreads) {
        const int g = i / a.D, d = i % a.D;
        float top = -INFINITY;
        for (int r = 0; r < blocks; ++r) top = fmaxf(top, *cl.map_shared_rank(&bm[g], r));
        const float base = top == -INFINITY ? 0.f : top;
        float x = 0.f, sum = 0.f;
        for (int r = 0; r < blocks; ++r) {
            const float f = exp2_fast(*cl.map_shared_rank(&bm[g], r) - base);
            x = fmaf(*cl.map_shared_rank(&bo[g][d], r), f, x);
            sum = fmaf(*cl.map_shared_rank(&bl[g], r), f, sum);
        }
        reinterpret_cast<T *>(a.o + b * a.ob + (h0 + g) * a.oh)[d] = from_f<T>(sum == 0.f ? 0.f : x / sum);
    }
    cl.sync();  // the others' sums stay until they are read
}

template <typename T, int LANES, int G, bool VEC> int launch(const AttnArgs &a, cudaStream_t st) {
    const int chunks = (a.group + G - 1) / G;
    const int64_t work = (int64_t)a.B * a.Hkv * chunks;
    // Blocks per sequence and group: enough for eight blocks on every SM, each
    // with 64 keys or more, at most 8 (a portable cluster)
    const int64_t keys = min((int64_t)a.T, (int64_t)a.window + a.sinks);
    int blocks = 1;
    while (blocks < 8 && work * blocks < 8 * (int64_t)sm_count() && keys >= blocks * 2 * 64) blocks *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1, a.Hkv * chunks, a.B);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    launch_clusters(cfg, 1, blocks, decode_kernel<T, LANES, G, VEC>, a);
    return launched("window attention decode");
}
template <typename T, int LANES, bool VEC> int by_group(const AttnArgs &a, cudaStream_t st) {
    if (a.group == 1) return launch<T, LANES, 1, VEC>(a, st);
    if (a.group == 2) return launch<T, LANES, 2, VEC>(a, st);
    if (a.group <= 4) return launch<T, LANES, 4, VEC>(a, st);
    return launch<T, LANES, 8, VEC>(a, st);
}
template <typename T, bool VEC> int by_size(const AttnArgs &a, cudaStream_t st) {
    constexpr int E = 16 / (int)sizeof(T);
    if (a.D <= 8 * E) return by_group<T, 8, VEC>(a, st);
    if (a.D <= 16 * E) return by_group<T, 16, VEC>(a, st);
    return by_group<T, 32, VEC>(a, st);  // 32-bit elements and D > 64
}
template <typename T> int run(const AttnArgs &a, bool vec, cudaStream_t st) {
    return vec ? by_size<T, true>(a, st) : by_size<T, false>(a, st);
}

}  // namespace
}  // namespace cailops

extern "C" int cail_ops_window_attention_decode(const cail_ops_attention_args *a, cail_ops_stream stream) {
    using namespace cailops;
    if (int rc = attn_check(a, false, "window attention decode")) return rc;
    if (!a->lengths) return fail(CAIL_OPS_EINVAL, "window attention decode: lengths are needed");
    if (a->B == 0) return CAIL_OPS_OK;
    if (tc_takes_decode(a)) return tc_decode(a, static_cast<cudaStream_t>(stream));
    const size_t s = type_size(a->type);
    const bool vec = a->D % (16 / s) == 0 && rows_aligned(a->q, a->B, 1, a->H, s, 16) &&
                     rows_aligned(a->k, a->B, a->T, a->Hkv, s, 16) && rows_aligned(a->v, a->B, a->T, a->Hkv, s, 16);
    const AttnArgs x = attn_args(a, false);
    auto st = static_cast<cudaStream_t>(stream);
    if (a->type == CAIL_OPS_F32) return run<float>(x, vec, st);
    if (a->type == CAIL_OPS_BF16) return run<__nv_bfloat16>(x, vec, st);
    return run<__half>(x, vec, st);
}
