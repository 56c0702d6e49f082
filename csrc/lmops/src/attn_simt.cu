// attn_simt.cu — window attention on the FP32 pipes: 32-bit inputs, and head
// sizes or strides that the tensor-core kernels do not take.
//
// Forward: a block owns 32 query rows of one head and goes once over the keys
// that some of them see (the sinks, then the window, side by side in tiles of
// 64), with the running maximum and sum of each row (16 threads share a row;
// each thread holds 4 rows x 4 columns of the scores and 4 rows x D/16 of the
// output).  Backward: p is recomputed from the kept log-sum; one kernel owns
// query rows and writes dq (and delta = do.o), the other owns keys, goes over
// the group's heads and the query rows that see them, and writes dk and dv.
// No atomics: results do not change from run to run.  Rows and keys at or
// beyond a sequence's length are never read, so what lies there may be
// anything.  Bound by the FP32 pipe and by reads of shared memory: 3 padded
// sequences of 333 tokens, 16 heads of 64, window 100 and 3 sinks, 21 us
// forward and 82 with the gradients; 2 x 2048, 16 heads, window 512, 251 us
// forward, 30 TFLOP/s.  4 x 4 rows and columns a thread: 4 x 8 measured the same.
#include "attn.cuh"

namespace cailops {
namespace {

constexpr int TR = 32;     // rows of a block, 4 threads' worth each
constexpr int kTile = 64;  // rows of the tiles that pass
constexpr float kNone = -INFINITY;

// rows of shared tiles are DP + 4 floats apart: 16-byte reads of 8 rows in a phase hit different banks
template <int DP> constexpr int ld() { return DP + 4; }
constexpr int kLdP = kTile + 4;

// ROWS rows of x, row r of the tile from row `row_of(r)` of x (rows below zero
// as zeros, columns >= D as zeros), as floats.  32-bit rows in whole vectors go
// by asynchronous copies (the caller commits and waits); the others through
// registers, all loads before the first store.
template <typename T, int DP, int ROWS, int THREADS, typename F>
__device__ __forceinline__ void load_tile(float *s, const char *base, int64_t st, F row_of, int D, bool vec) {
    constexpr int N = 16 / (int)sizeof(T), C = DP / N, ITER = ROWS * C / THREADS;
    static_assert(ROWS * C % THREADS == 0);
    if (vec && sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < ITER; ++k) {
            const int i = threadIdx.x + k * THREADS, r = i / C, c = (i % C) * N, from = row_of(r);
            const bool in = from >= 0 && c < D;
            const char *src = in ? base + (int64_t)from * st + c * sizeof(T) : base;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(s + r * ld<DP>() + c)), "l"(src),
                         "r"(in ? 16 : 0)
                         : "memory");
        }
    } else if (vec) {
        Vec<T, N> x[ITER];
#pragma unroll
        for (int k = 0; k < ITER; ++k) {
            const int i = threadIdx.x + k * THREADS, r = i / C, c = (i % C) * N, from = row_of(r);
            if (from >= 0 && c < D) x[k] = *reinterpret_cast<const Vec<T, N> *>(base + (int64_t)from * st + c * sizeof(T));
        }
#pragma unroll
        for (int k = 0; k < ITER; ++k) {
            const int i = threadIdx.x + k * THREADS, r = i / C, c = (i % C) * N;
            const bool in = row_of(r) >= 0 && c < D;
#pragma unroll
            for (int e = 0; e < N; ++e) s[r * ld<DP>() + c + e] = in ? to_f(x[k].v[e]) : 0.f;
        }
    } else {
#pragma unroll 4
        for (int i = threadIdx.x; i < ROWS * DP; i += THREADS) {
            const int r = i / DP, c = i % DP, from = row_of(r);
            const bool in = from >= 0 && c < D;
            s[r * ld<DP>() + c] = in ? to_f(*reinterpret_cast<const T *>(base + (int64_t)from * st + c * sizeof(T))) : 0.f;
        }
    }
}
// rows r0 .. of a sequence that ends at n
struct From {
    int r0, n;
    __device__ __forceinline__ int operator()(int r) const { return r0 + r < n ? r0 + r : -1; }
};
// The keys that the query rows [i0, i1) of a sequence of n tokens need: the
// sinks before the window, then the window, side by side in tiles, so that a
// few sinks take a few rows of a tile and no tile starts before the window.
struct Keys {
    int sinks, first, total, count;
    __device__ __forceinline__ Keys(int i0, int i1, int n, int window, int all_sinks) {
        i1 = min(i1, n);
        first = window > i0 ? 0 : i0 - window + 1;
        sinks = min(all_sinks, first);
        total = i0 < i1 ? sinks + i1 - first : 0;
        count = (total + kTile - 1) / kTile;
    }
    // the key in place x (a key behind the last row where x is behind the last place)
    __device__ __forceinline__ int key(int x) const { return x < sinks ? x : x - sinks + first; }
};
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// acc[r][c] = sum_d x[ty*4+r][d] * y[tx+16c][d] for c < C, even and odd d apart until the end
template <int DP, int C> __device__ __forceinline__ void dot_columns(const float *x, const float *y, float acc[4][4], int ty, int tx) {
    uint64_t acc2[4][C] = {};
#pragma unroll 4
    for (int d = 0; d < DP; d += 4) {
        ulonglong2 a[4], b[C];
#pragma unroll
        for (int r = 0; r < 4; ++r) a[r] = *reinterpret_cast<const ulonglong2 *>(x + (ty * 4 + r) * ld<DP>() + d);
#pragma unroll
        for (int c = 0; c < C; ++c) b[c] = *reinterpret_cast<const ulonglong2 *>(y + (tx + 16 * c) * ld<DP>() + d);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < C; ++c) acc2[r][c] = fma_two(a[r].y, b[c].y, fma_two(a[r].x, b[c].x, acc2[r][c]));
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float e, o;
            apart(acc2[r][c], e, o);
            acc[r][c] = e + o;
        }
}

// the same for the first `valid` rows of y, in halves (what lies behind is left zero)
template <int DP> __device__ __forceinline__ void dot_tile(const float *x, const float *y, float acc[4][4], int ty, int tx, int valid) {
    if (valid > kTile / 2) {
        dot_columns<DP, 4>(x, y, acc, ty, tx);
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r][2] = acc[r][3] = 0.f;
        dot_columns<DP, 2>(x, y, acc, ty, tx);
    }
}

// column c of a thread's DP/16 output columns
template <int DP> __device__ __forceinline__ int column(int tx, int c) {
    constexpr int NC = DP / 16;
    if constexpr (NC <= 4) return tx * NC + c;
    return (c / 4) * 64 + tx * 4 + c % 4;
}
// a thread's columns in pairs: [r][NC / 2]
template <int DP> struct Out {
    static constexpr int NP = DP / 32;
    uint64_t v[4][NP];
    __device__ __forceinline__ Out() {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < NP; ++c) v[r][c] = 0;
    }
    __device__ __forceinline__ void scale(int r, float f) {
#pragma unroll
        for (int c = 0; c < NP; ++c) v[r][c] = mul_two(v[r][c], two(f, f));
    }
    __device__ __forceinline__ float at(int r, int c) const {
        float lo, hi;
        apart(v[r][c / 2], lo, hi);
        return c % 2 ? hi : lo;
    }
};
template <int DP> __device__ __forceinline__ void row_of(const float *y, uint64_t *w, int tx) {
    if constexpr (DP == 32) {
        w[0] = *reinterpret_cast<const uint64_t *>(y + tx * 2);
    } else {
#pragma unroll
        for (int g = 0; g < DP / 64; ++g) {
            const ulonglong2 f = *reinterpret_cast<const ulonglong2 *>(y + g * 64 + tx * 4);
            w[g * 2] = f.x, w[g * 2 + 1] = f.y;
        }
    }
}
// o[r][:] += sum_j p[ty*4+r][j] * y[j][:], over four j
template <int DP> __device__ __forceinline__ void out_four(const float *p, const float *y, Out<DP> &o, int ty, int tx, int j) {
    float4 a[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) a[r] = *reinterpret_cast<const float4 *>(p + (ty * 4 + r) * kLdP + j);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        uint64_t w[Out<DP>::NP];
        row_of<DP>(y + (j + e) * ld<DP>(), w, tx);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float f = e == 0 ? a[r].x : e == 1 ? a[r].y : e == 2 ? a[r].z : a[r].w;
#pragma unroll
            for (int c = 0; c < Out<DP>::NP; ++c) o.v[r][c] = fma_two(two(f, f), w[c], o.v[r][c]);
        }
    }
}
// over the first `valid` j, in fours; all of them, unrolled, where few are left out (p is zero behind them)
template <int DP> __device__ __forceinline__ void out_tile(const float *p, const float *y, Out<DP> &o, int ty, int tx, int valid) {
    if (valid > kTile * 3 / 4) {
#pragma unroll 4
        for (int j = 0; j < kTile; j += 4) out_four<DP>(p, y, o, ty, tx, j);
    } else {
#pragma unroll 1
        for (int j = 0; j < valid; j += 4) out_four<DP>(p, y, o, ty, tx, j);
    }
}

__device__ __forceinline__ float half_max(float x) {
#pragma unroll
    for (int o = 8; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}
__device__ __forceinline__ float half_sum(float x) {
#pragma unroll
    for (int o = 8; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

template <typename T, int DP>
__global__ void __launch_bounds__(TR * 4) simt_forward(const AttnArgs a, bool vec) {
    constexpr int NC = DP / 16;
    extern __shared__ float4 smem4[];
    constexpr int TILE = kTile * ld<DP>();
    float *sq = reinterpret_cast<float *>(smem4), *sk = sq + TR * ld<DP>(), *sv = sk + TILE, *sp = sv + TILE;
    const int h = blockIdx.y, b = blockIdx.z, hk = h / a.group;
    const int i0 = (gridDim.x - 1 - blockIdx.x) * TR;  // the longest rows first
    const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16;
    const int n = length_of(a, b);
    const Keys keys(i0, i0 + TR, n, a.window, a.sinks);
    const char *kp = a.k + b * a.kb + hk * a.kh, *vp = a.v + b * a.vb + hk * a.vh;

    load_tile<T, DP, TR, TR * 4>(sq, a.q + b * a.qb + h * a.qh, a.qt, From{i0, n}, a.D, vec);
    Out<DP> o;
    float m[4], l[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) m[r] = kNone, l[r] = 0.f;

    auto fetch = [&](float *s, const char *from, int64_t st, int x) {
        load_tile<T, DP, kTile, TR * 4>(s, from, st, [&](int r) { return x * kTile + r < keys.total ? keys.key(x * kTile + r) : -1; }, a.D, vec);
        copies_issued();
    };
    fetch(sk, kp, a.kt, 0);
    for (int x = 0; x < keys.count; ++x) {
        const int valid = keys.total - x * kTile;
        copies_done<0>();
        __syncthreads();  // the keys are there, the values' place is free
        fetch(sv, vp, a.vt, x);
        float s[4][4];
        dot_tile<DP>(sq, sk, s, ty, tx, valid);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = i0 + ty * 4 + r;
            float top = kNone;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                s[r][c] = seen(i, keys.key(x * kTile + tx + 16 * c), n, a.window, a.sinks) ? s[r][c] * a.scale_log2 : kNone;
                top = fmaxf(top, s[r][c]);
            }
            top = fmaxf(m[r], half_max(top));
            const float base = top == kNone ? 0.f : top, turn = exp2_fast(m[r] - base);
            m[r] = top;
            float sum = 0.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float p = exp2_fast(s[r][c] - base);
                sum += p;
                sp[(ty * 4 + r) * kLdP + tx + 16 * c] = p;
            }
            l[r] = l[r] * turn + half_sum(sum);
            o.scale(r, turn);
        }
        copies_done<0>();
        __syncthreads();  // the values are there, the keys' place is free
        if (x + 1 < keys.count) fetch(sk, kp, a.kt, x + 1);
        out_tile<DP>(sp, sv, o, ty, tx, valid);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int i = i0 + ty * 4 + r;
        if (i >= a.T) continue;
        const float inv = l[r] > 0.f ? 1.f / l[r] : 0.f;
        T *out = reinterpret_cast<T *>(a.o + b * a.ob + (int64_t)i * a.ot + h * a.oh);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = column<DP>(tx, c);
            const float f = l[r] == 0.f ? 0.f : o.at(r, c) * inv;
            if (d >= a.D) continue;
            out[d] = from_f<T>(f);
            if (sizeof(T) == 2 && i < a.rest_rows) reinterpret_cast<T *>(a.rest + b * a.rb + (int64_t)i * a.rt + h * a.rh)[d] = from_f<T>(rest_of<T>(f));
        }
        if (a.lse && tx == 0) a.lse[((int64_t)b * a.H + h) * a.lse_row + i] = l[r] == 0.f ? 0.f : m[r] + log2f(l[r]);
    }
}

// dq and delta of a block's query rows
template <typename T, int DP>
__global__ void __launch_bounds__(TR * 4) simt_dq(const AttnArgs a, bool vec) {
    constexpr int NC = DP / 16;
    constexpr int TILE = kTile * ld<DP>();
    extern __shared__ float4 smem4[];
    float *sq = reinterpret_cast<float *>(smem4), *sg = sq + TR * ld<DP>(), *sk = sg + TR * ld<DP>(), *sv = sk + TILE, *sp = sv + TILE;
    const int h = blockIdx.y, b = blockIdx.z, hk = h / a.group;
    const int i0 = (gridDim.x - 1 - blockIdx.x) * TR;
    const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16;
    const int n = length_of(a, b);
    const Keys keys(i0, i0 + TR, n, a.window, a.sinks);
    const char *kp = a.k + b * a.kb + hk * a.kh, *vp = a.v + b * a.vb + hk * a.vh;

    auto fetch = [&](float *s, const char *from, int64_t st, int x) {
        load_tile<T, DP, kTile, TR * 4>(s, from, st, [&](int r) { return x * kTile + r < keys.total ? keys.key(x * kTile + r) : -1; }, a.D, vec);
        copies_issued();
    };
    // o, and what rounding took from it, pass through the keys' place
    float *so = sk, *srest = sk + TR * ld<DP>();
    static_assert(2 * TR <= kTile);
    const From rows = {i0, n};
    load_tile<T, DP, TR, TR * 4>(sq, a.q + b * a.qb + h * a.qh, a.qt, rows, a.D, vec);
    load_tile<T, DP, TR, TR * 4>(sg, a.dout + b * a.gb + h * a.gh, a.gt, rows, a.D, vec);
    load_tile<T, DP, TR, TR * 4>(so, a.o + b * a.ob + h * a.oh, a.ot, rows, a.D, vec);
    const bool rest = sizeof(T) == 2 && i0 < a.rest_rows;
    if (rest) load_tile<T, DP, TR, TR * 4>(srest, a.rest + b * a.rb + h * a.rh, a.rt, From{i0, min(n, a.rest_rows)}, a.D, vec);
    copies_issued();
    fetch(sv, vp, a.vt, 0);
    copies_done<1>();
    __syncthreads();
    float delta[4], lse[4];
    Out<DP> dq;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int row = ty * 4 + r, i = i0 + row;
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int at = row * ld<DP>() + tx + 16 * c;
            s = fmaf(sg[at], rest ? so[at] + srest[at] : so[at], s);
        }
        delta[r] = half_sum(s);
        const int64_t at = ((int64_t)b * a.H + h) * a.lse_row + i;
        lse[r] = i < n ? a.lse[at] : 0.f;
        if (i < a.T && tx == 0) a.delta[at] = delta[r];
    }
    for (int x = 0; x < keys.count; ++x) {
        const int valid = keys.total - x * kTile;
        copies_done<0>();
        __syncthreads();  // the values are there, the keys' place is free
        fetch(sk, kp, a.kt, x);
        float s[4][4], dp[4][4];
        dot_tile<DP>(sg, sv, dp, ty, tx, valid);
        copies_done<0>();
        __syncthreads();  // the keys are there, the values' place is free
        if (x + 1 < keys.count) fetch(sv, vp, a.vt, x + 1);
        dot_tile<DP>(sq, sk, s, ty, tx, valid);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int i = i0 + ty * 4 + r;
                const bool on = seen(i, keys.key(x * kTile + tx + 16 * c), n, a.window, a.sinks) && !one_key(i, a.window, a.sinks);
                sp[(ty * 4 + r) * kLdP + tx + 16 * c] = on ? exp2_fast(fmaf(s[r][c], a.scale_log2, -lse[r])) * (dp[r][c] - delta[r]) : 0.f;
            }
        __syncwarp();
        out_tile<DP>(sp, sk, dq, ty, tx, valid);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int i = i0 + ty * 4 + r;
        if (i >= a.T) continue;
        T *out = reinterpret_cast<T *>(a.dq + b * a.dqb + (int64_t)i * a.dqt + h * a.dqh);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = column<DP>(tx, c);
            if (d < a.D) out[d] = from_f<T>(dq.at(r, c) * a.scale);
        }
    }
}

// dk and dv of a block's keys, over the group's heads and the query rows that see them
template <typename T, int DP>
__global__ void __launch_bounds__(TR * 4) simt_dkv(const AttnArgs a, bool vec, const SinkParts parts) {
    constexpr int NC = DP / 16;
    constexpr int TILE = kTile * ld<DP>();
    extern __shared__ float4 smem4[];
    float *sk = reinterpret_cast<float *>(smem4), *sv = sk + TR * ld<DP>(), *sq = sv + TR * ld<DP>(), *sg = sq + TILE, *sp = sg + TILE,
          *sd = sp + TR * kLdP;
    __shared__ float row_lse[kTile], row_delta[kTile];
    const int hk = blockIdx.y, b = blockIdx.z;
    int tile = blockIdx.x, split = 0;
    const bool parted = parts.splits > 1 && tile < parts.tiles * parts.splits;
    if (parted) split = tile % parts.splits, tile /= parts.splits;
    else if (parts.splits > 1) tile -= parts.tiles * (parts.splits - 1);
    const int j0 = tile * TR;
    const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16;
    const int n = length_of(a, b);
    int begin, end;
    query_range(j0, j0 + TR, n, a.window, a.sinks, begin, end);
    load_tile<T, DP, TR, TR * 4>(sk, a.k + b * a.kb + hk * a.kh, a.kt, From{j0, n}, a.D, vec);
    load_tile<T, DP, TR, TR * 4>(sv, a.v + b * a.vb + hk * a.vh, a.vt, From{j0, n}, a.D, vec);
    Out<DP> dk, dv;
    // the tiles that pass: the group's heads in turn, each over the rows that see these keys
    const int per = end > begin ? (end - begin + kTile - 1) / kTile : 0;
    int first = 0, count = a.group * per;
    if (parted) {  // this part of them
        const int share = (count + parts.splits - 1) / parts.splits;
        first = min(count, split * share);
        count = min(count, first + share);
    }
    auto rows = [&](int x) { return begin + x % per * kTile; };
    auto fetch_g = [&](int x) {
        load_tile<T, DP, kTile, TR * 4>(sg, a.dout + b * a.gb + (hk * a.group + x / per) * a.gh, a.gt, From{rows(x), n}, a.D, vec);
        copies_issued();
    };
    auto fetch_q = [&](int x) {
        const int h = hk * a.group + x / per, i0 = rows(x);
        load_tile<T, DP, kTile, TR * 4>(sq, a.q + b * a.qb + h * a.qh, a.qt, From{i0, n}, a.D, vec);
        if (tid < kTile) {
            const int64_t row = ((int64_t)b * a.H + h) * a.lse_row + i0 + tid;
            row_lse[tid] = i0 + tid < n ? a.lse[row] : 0.f;
            row_delta[tid] = i0 + tid < n ? a.delta[row] : 0.f;
        }
        copies_issued();
    };
    if (first < count) fetch_g(first);
    for (int x = first; x < count; ++x) {
        const int i0 = rows(x), valid = end - i0;
        copies_done<0>();
        __syncthreads();  // do is there, q's place is free
        fetch_q(x);
        float s[4][4], dp[4][4];
        dot_tile<DP>(sv, sg, dp, ty, tx, valid);
        copies_done<0>();
        __syncthreads();  // q is there
        dot_tile<DP>(sk, sq, s, ty, tx, valid);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int i = tx + 16 * c;
                const bool on = seen(i0 + i, j0 + ty * 4 + r, n, a.window, a.sinks);
                const float p = on ? exp2_fast(fmaf(s[r][c], a.scale_log2, -row_lse[i])) : 0.f;
                sp[(ty * 4 + r) * kLdP + i] = p;
                sd[(ty * 4 + r) * kLdP + i] = on && !one_key(i0 + i, a.window, a.sinks) ? p * (dp[r][c] - row_delta[i]) : 0.f;
            }
        __syncwarp();
        out_tile<DP>(sp, sg, dv, ty, tx, valid);
        __syncthreads();  // do's place is free
        if (x + 1 < count) fetch_g(x + 1);
        out_tile<DP>(sd, sq, dk, ty, tx, valid);
    }
    if (parted) {
        float *sums = parts.sums + ((((int64_t)b * a.Hkv + hk) * parts.tiles + tile) * parts.splits + split) * (2 * TR * DP);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int at = (ty * 4 + r) * DP + column<DP>(tx, c);
                sums[at] = dk.at(r, c) * a.scale, sums[TR * DP + at] = dv.at(r, c);
            }
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int j = j0 + ty * 4 + r;
        if (j >= a.T) continue;
        T *ok = reinterpret_cast<T *>(a.dk + b * a.dkb + (int64_t)j * a.dkt + hk * a.dkh);
        T *ov = reinterpret_cast<T *>(a.dv + b * a.dvb + (int64_t)j * a.dvt + hk * a.dvh);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = column<DP>(tx, c);
            if (d < a.D) ok[d] = from_f<T>(dk.at(r, c) * a.scale), ov[d] = from_f<T>(dv.at(r, c));
        }
    }
}

template <typename K> int prepare(K kernel, size_t smem) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    return e == cudaSuccess ? CAIL_OPS_OK : fail(CAIL_OPS_ECUDA, "window attention: %s", cudaGetErrorString(e));
}

// 32 rows a block and one place each for the keys and the values, whose loads
// pass under the other's products: four blocks of four warps per SM forward,
// three backward.  (64 rows and two places of each, two blocks of eight warps:
// 2 x 2048 tokens, 16 heads of 64, window 512, forward and backward 1214 us
// instead of 1071; 2 x 4096, 8 heads, window 250, 718 instead of 632, window 8,
// 310 instead of 148.)
template <typename T, int DP> int forward(const AttnArgs &a, bool vec, cudaStream_t st) {
    const size_t smem = (TR * ld<DP>() + 2 * kTile * ld<DP>() + TR * kLdP) * sizeof(float);
    if (int rc = prepare(simt_forward<T, DP>, smem)) return rc;
    simt_forward<T, DP><<<dim3((a.T + TR - 1) / TR, a.H, a.B), TR * 4, smem, st>>>(a, vec);
    return launched("window attention");
}
template <typename T, int DP> int backward(const AttnArgs &a, const SinkParts &parts, bool vec, cudaStream_t st) {
    const unsigned tiles = (a.T + TR - 1) / TR;
    size_t smem = (2 * TR * ld<DP>() + 2 * kTile * ld<DP>() + TR * kLdP) * sizeof(float);
    if (int rc = prepare(simt_dq<T, DP>, smem)) return rc;
    simt_dq<T, DP><<<dim3(tiles, a.H, a.B), TR * 4, smem, st>>>(a, vec);
    if (int rc = launched("window attention backward")) return rc;
    smem += TR * kLdP * sizeof(float);
    if (int rc = prepare(simt_dkv<T, DP>, smem)) return rc;
    simt_dkv<T, DP><<<dim3(tiles + parts.tiles * (parts.splits - 1), a.Hkv, a.B), TR * 4, smem, st>>>(a, vec, parts);
    if (int rc = launched("window attention backward")) return rc;
    return parts.splits > 1 ? join<T, DP, TR>(a, parts, st) : CAIL_OPS_OK;
}
SinkParts parts_of(const cail_ops_attention_args *a) { return sink_parts(a, TR, kTile, 3 * (int64_t)sm_count()); }
int padded(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }
template <typename T, int DP> int sized(const AttnArgs &a, const SinkParts &parts, bool vec, bool back, cudaStream_t st) {
    return back ? backward<T, DP>(a, parts, vec, st) : forward<T, DP>(a, vec, st);
}
template <typename T> int run(const cail_ops_attention_args *c, bool vec, bool back, cudaStream_t st) {
    const AttnArgs a = attn_args(c, back);
    SinkParts parts = {1, 0, nullptr};
    if (back) {
        parts = parts_of(c);
        const size_t bytes = sink_bytes(c, parts, TR, padded(a.D));
        if (c->workspace_bytes < bytes || (bytes && (!c->workspace || !aligned(c->workspace, 16))))
            return fail(CAIL_OPS_EINVAL, "window attention backward: a workspace of %zu bytes is needed", bytes);
        parts.sums = static_cast<float *>(c->workspace);
    }
    if (a.D <= 32) return sized<T, 32>(a, parts, vec, back, st);
    if (a.D <= 64) return sized<T, 64>(a, parts, vec, back, st);
    return sized<T, 128>(a, parts, vec, back, st);
}

}  // namespace

// so many parts that none is longer than a key tile without sinks or than a
// block's share of all tiles, whichever is more; no more tiles in all than a grid has
SinkParts sink_parts(const cail_ops_attention_args *c, int rows, int stream, int64_t slots) {
    SinkParts none = {1, 0, nullptr};
    if (c->sinks == 0 || c->window >= c->T) return none;
    const int64_t group = c->H / c->Hkv, tiles = ((int64_t)c->T + rows - 1) / rows, q_tiles = ((int64_t)c->T + stream - 1) / stream;
    const int64_t sink_tiles = ((int64_t)(c->sinks < c->T ? c->sinks : c->T) + rows - 1) / rows;
    const int64_t plain = group * (((int64_t)c->window + rows) / stream + 1), sunk = group * q_tiles;
    if (sunk <= plain) return none;
    const int64_t all = (int64_t)c->B * c->Hkv * ((tiles - sink_tiles) * plain + sink_tiles * sunk);
    const int64_t share = all / slots > plain ? all / slots : plain;
    int64_t splits = (sunk + share - 1) / share;
    if (splits > 32) splits = 32;
    if (tiles <= kMostTiles && splits > 1 + (kMostTiles - tiles) / sink_tiles) splits = 1 + (kMostTiles - tiles) / sink_tiles;
    if (splits <= 1) return none;
    return {(int)splits, (int)sink_tiles, nullptr};
}

int attn_check(const cail_ops_attention_args *a, bool backward, const char *who) {
    if (a->type < CAIL_OPS_F32 || a->type > CAIL_OPS_F16) return fail(CAIL_OPS_EINVAL, "%s: unknown element type %d", who, a->type);
    if (a->B < 0 || a->T < 0 || a->H < 1 || a->Hkv < 1 || a->H % a->Hkv || a->D < 1 || a->D > 128)
        return fail(CAIL_OPS_EINVAL, "%s: bad sizes (B %d T %d H %d Hkv %d D %d)", who, a->B, a->T, a->H, a->Hkv, a->D);
    if (a->B > 65535 || a->H > 65535) return fail(CAIL_OPS_EINVAL, "%s: at most 65535 sequences and heads", who);
    if (a->T > (1 << 30)) return fail(CAIL_OPS_EINVAL, "%s: at most 2^30 tokens", who);
    if (a->window < 1 || a->sinks < 0) return fail(CAIL_OPS_EINVAL, "%s: window %d and sinks %d", who, a->window, a->sinks);
    if (a->o_rest.ptr && (a->rest_rows < 0 || a->rest_rows > a->T))
        return fail(CAIL_OPS_EINVAL, "%s: the rest of %d rows of %d", who, a->rest_rows, a->T);
    if (backward && (!a->lse || !a->delta)) return fail(CAIL_OPS_EINVAL, "%s: lse and delta are needed", who);
    return CAIL_OPS_OK;
}

AttnArgs attn_args(const cail_ops_attention_args *a, bool backward) {
    const int64_t s = (int64_t)type_size(a->type);
    AttnArgs x = {};
    x.B = a->B, x.T = a->T, x.H = a->H, x.Hkv = a->Hkv, x.D = a->D, x.group = a->H / a->Hkv;
    x.window = a->window, x.sinks = a->sinks;
    x.scale = a->scale, x.scale_log2 = a->scale * kLog2e;
    x.lengths = a->lengths;
    x.q = static_cast<const char *>(a->q.ptr), x.qb = a->q.sb * s, x.qt = a->q.st * s, x.qh = a->q.sh * s;
    x.k = static_cast<const char *>(a->k.ptr), x.kb = a->k.sb * s, x.kt = a->k.st * s, x.kh = a->k.sh * s;
    x.v = static_cast<const char *>(a->v.ptr), x.vb = a->v.sb * s, x.vt = a->v.st * s, x.vh = a->v.sh * s;
    x.o = static_cast<char *>(a->o.ptr), x.ob = a->o.sb * s, x.ot = a->o.st * s, x.oh = a->o.sh * s;
    x.fine_rows = cail_ops_rest_rows(a->T, a->D, a->window, a->sinks);
    if (a->type != CAIL_OPS_F32 && a->o_rest.ptr) {
        x.rest = static_cast<char *>(a->o_rest.ptr), x.rb = a->o_rest.sb * s, x.rt = a->o_rest.st * s, x.rh = a->o_rest.sh * s;
        x.rest_rows = a->rest_rows;
    }
    x.lse = a->lse, x.lse_row = (a->T + 3) / 4 * 4;
    if (backward) {
        x.dout = static_cast<const char *>(a->dout.ptr), x.gb = a->dout.sb * s, x.gt = a->dout.st * s, x.gh = a->dout.sh * s;
        x.dq = static_cast<char *>(a->dq.ptr), x.dqb = a->dq.sb * s, x.dqt = a->dq.st * s, x.dqh = a->dq.sh * s;
        x.dk = static_cast<char *>(a->dk.ptr), x.dkb = a->dk.sb * s, x.dkt = a->dk.st * s, x.dkh = a->dk.sh * s;
        x.dv = static_cast<char *>(a->dv.ptr), x.dvb = a->dv.sb * s, x.dvt = a->dv.st * s, x.dvh = a->dv.sh * s;
        x.delta = a->delta;
    }
    return x;
}

}  // namespace cailops

using namespace cailops;

static bool attn_vectors(const cail_ops_attention_args *a, bool backward) {
    const size_t s = type_size(a->type);
    return a->D % (16 / s) == 0 && rows_aligned(a->q, a->B, a->T, a->H, s, 16) && rows_aligned(a->k, a->B, a->T, a->Hkv, s, 16) &&
           rows_aligned(a->v, a->B, a->T, a->Hkv, s, 16) &&
           (!backward || ((!a->o_rest.ptr || rows_aligned(a->o_rest, a->B, a->rest_rows, a->H, s, 16)) && rows_aligned(a->o, a->B, a->T, a->H, s, 16) && rows_aligned(a->dout, a->B, a->T, a->H, s, 16)));
}

extern "C" int cail_ops_window_attention(const cail_ops_attention_args *a, cail_ops_stream stream) {
    if (int rc = attn_check(a, false, "window attention")) return rc;
    if (a->B == 0 || a->T == 0) return CAIL_OPS_OK;
    auto st = static_cast<cudaStream_t>(stream);
    if (tc_takes(a)) return tc_forward(a, st);
    const bool vec = attn_vectors(a, false);
    if (a->type == CAIL_OPS_F32) return run<float>(a, vec, false, st);
    if (a->type == CAIL_OPS_BF16) return run<__nv_bfloat16>(a, vec, false, st);
    return run<__half>(a, vec, false, st);
}

extern "C" size_t cail_ops_window_attention_workspace(const cail_ops_attention_args *a) {
    if (attn_check(a, true, "window attention backward") || a->B == 0 || a->T == 0) return 0;
    return tc_takes_backward(a) ? tc_workspace(a) : sink_bytes(a, parts_of(a), TR, padded(a->D));
}

extern "C" int cail_ops_window_attention_backward(const cail_ops_attention_args *a, cail_ops_stream stream) {
    if (int rc = attn_check(a, true, "window attention backward")) return rc;
    if (a->B == 0 || a->T == 0) return CAIL_OPS_OK;
    auto st = static_cast<cudaStream_t>(stream);
    if (tc_takes_backward(a)) return tc_backward(a, st);
    const bool vec = attn_vectors(a, true);
    if (a->type == CAIL_OPS_F32) return run<float>(a, vec, true, st);
    if (a->type == CAIL_OPS_BF16) return run<__nv_bfloat16>(a, vec, true, st);
    return run<__half>(a, vec, true, st);
}
