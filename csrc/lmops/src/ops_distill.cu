// ops_distill.cu — distillation from a teacher's top logits, with the hard
// labels' cross entropy beside it: forward, and the gradient of the logits.
//
// With q = softmax(z / tau) over the vocabulary and p = softmax(t / tau) over
// the teacher's K entries of a row, the row's loss is
//   L = (1 - w) tau^2 sum_k p_k (log p_k - log q_id(k)) + w (lse(z) - z_y)
// and its gradient
//   dL/dz_j = (1 - w) tau (q_j sum_k p_k - sum_{k: id(k) = j} p_k)
//             + w (softmax(z)_j - [j = y]).
// Forward reads a row once, keeping a running maximum m and the sums of
// exp(z - m) and exp((z - m) / tau); a row is shared by a cluster of up to 8
// blocks that join over distributed shared memory, so a few rows still use
// the whole GPU.  Backward reads the row again and writes its gradient; the
// K + 1 entries with a teacher or label term are written after the rest of
// the row by the block that owns them.  Everything is summed in a fixed
// order: results do not change from run to run.
//
// Bound by latency for a few rows (37 x 50257 float32: 22 us forward and
// backward, 15 MB).  Rows for every SM go through rings of bulk copies
// (distill_ring_kernel, distill_backward_ring_kernel).
#include <cooperative_groups.h>

#include "tc.cuh"

namespace cg = cooperative_groups;

namespace cailops {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;

// what forward keeps of a row: [0] m, [1] sum exp(z - m), [2] sum exp((z - m) / tau),
// [3] the teacher's maximum, [4] 1 / sum exp((t - max) / tau) (0: no teacher entry), [5] 1 if the row counts
constexpr int kStats = 8;

struct Args {
    int64_t N, V, ldz, ldg;
    const void *z;
    void *grad;
    const void *ids, *teacher;
    const int64_t *targets;
    const float *grad_loss, *factor;
    float *rows, *stats;
    int K, ids64, teacher_type, per_row_grad;
    float inv_tau, tau, hard;
};

__device__ __forceinline__ int64_t id_at(const Args &a, int64_t i) {
    return a.ids64 ? static_cast<const int64_t *>(a.ids)[i] : (int64_t) static_cast<const int32_t *>(a.ids)[i];
}
__device__ __forceinline__ float teacher_at(const Args &a, int64_t i) {
    if (a.teacher_type == CAIL_OPS_F32) return static_cast<const float *>(a.teacher)[i];
    if (a.teacher_type == CAIL_OPS_BF16) return to_f(static_cast<const __nv_bfloat16 *>(a.teacher)[i]);
    return to_f(static_cast<const __half *>(a.teacher)[i]);
}

// 16 bytes of a row as pairs of floats, and the running maximum of such
// vectors (NaN aside), kept packed for the 16-bit types
template <typename T> struct Pairs {
    static constexpr int count = 8 / (int)sizeof(T);
    uint64_t x[count];
    __device__ __forceinline__ explicit Pairs(const uint4 &u);
};
template <> __device__ __forceinline__ Pairs<float>::Pairs(const uint4 &u) {
    x[0] = two(__uint_as_float(u.x), __uint_as_float(u.y)), x[1] = two(__uint_as_float(u.z), __uint_as_float(u.w));
}
template <> __device__ __forceinline__ Pairs<__nv_bfloat16>::Pairs(const uint4 &u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = two(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
template <> __device__ __forceinline__ Pairs<__half>::Pairs(const uint4 &u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        x[i] = two(f.x, f.y);
    }
}
template <int U> __device__ __forceinline__ float top_of(const uint4 (&u)[U], float) {
    float t = -INFINITY;
#pragma unroll
    for (int k = 0; k < U; ++k)
        t = fmaxf(t, fmaxf(fmaxf(__uint_as_float(u[k].x), __uint_as_float(u[k].y)), fmaxf(__uint_as_float(u[k].z), __uint_as_float(u[k].w))));
    return t;
}
template <typename H2, int U> __device__ __forceinline__ H2 packed_top(const uint4 (&u)[U]) {
    auto h = [](const uint32_t &w) { return *reinterpret_cast<const H2 *>(&w); };
    H2 t = __hmax2(__hmax2(h(u[0].x), h(u[0].y)), __hmax2(h(u[0].z), h(u[0].w)));
#pragma unroll
    for (int k = 1; k < U; ++k) t = __hmax2(t, __hmax2(__hmax2(h(u[k].x), h(u[k].y)), __hmax2(h(u[k].z), h(u[k].w))));
    return t;
}
template <int U> __device__ __forceinline__ float top_of(const uint4 (&u)[U], __nv_bfloat16) {
    const __nv_bfloat162 t = packed_top<__nv_bfloat162>(u);
    return fmaxf(__low2float(t), __high2float(t));
}
template <int U> __device__ __forceinline__ float top_of(const uint4 (&u)[U], __half) {
    const __half2 t = packed_top<__half2>(u);
    return fmaxf(__low2float(t), __high2float(t));
}

// MODE of the sums: which of exp(z - m) and exp((z - m) / tau) are needed.
// kSquare: both with tau = 2, where the first is the second squared.
enum { kOne, kSquare, kBoth };

// exp((x - m) / tau) is taken as exp2((x - m) c): the difference first, as
// softmax does not depend on what is common to a row and neither may its
// rounding.  (c x - c m is one instruction instead of two, but off by the
// rounding of c m: 1e-3 in the loss of logits around 1e4.  Forward over 8192 x
// 50257 bf16, tau 2: 155 us, and 158 that way.)
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

// m is a reference, not always the maximum: it moves only when a value lies so
// far above it (a factor of 2^40 in a sum) that the sums could leave 32 bits'
// range.
template <int MODE> struct Sums {
    float m = -INFINITY, s1 = 0.f, st = 0.f;
    // kOne keeps one sum, st, at the scale `c` (log2(e) / tau, or log2(e) for the label alone)
    __device__ __forceinline__ void scale_to(float n, float c) {  // n >= m
        if (n == m) return;
        const float d = m - n;  // minus infinity while nothing is summed: sums of 0 stay 0, NaN stays
        const float e = exp2_fast(d * c);
        st *= e;
        if (MODE == kSquare) s1 *= e * e;
        if (MODE == kBoth) s1 *= exp2_fast(d * kLog2e);
        m = n;
    }
    __device__ __forceinline__ void join(float om, float os1, float ost, float c) {
        Sums o;
        o.m = om, o.s1 = os1, o.st = ost;
        const float n = fmaxf(m, om);
        scale_to(n, c);
        o.scale_to(n, c);
        s1 += o.s1, st += o.st;
    }
};
// The sums while a thread goes through its part of a row: two packed sums each.
template <int MODE> struct Running {
    float c, reach;          // reach: how far above the reference a value may lie
    float m = -INFINITY, limit = -INFINITY;
    uint64_t minus = 0;      // minus the reference
    uint64_t t2[2] = {0, 0}, q2[2] = {0, 0};
    __device__ __forceinline__ explicit Running(float c_) : c(c_) {
        const float steepest = MODE == kOne ? c : fmaxf(c, kLog2e);
        reach = (MODE == kSquare ? 20.f / c : 40.f / steepest);
    }
    __device__ __forceinline__ Sums<MODE> sums() const {
        Sums<MODE> s;
        float a0, a1;
        s.m = m;
        apart(add_two(t2[0], t2[1]), a0, a1);
        s.st = a0 + a1;
        apart(add_two(q2[0], q2[1]), a0, a1);
        s.s1 = a0 + a1;
        return s;
    }
    __device__ __forceinline__ void move_to(float top) {
        Sums<MODE> s = sums();
        s.scale_to(top, c);
        m = top, limit = top + reach;
        minus = two(-base_of(m), -base_of(m));
        t2[0] = two(s.st, 0.f), t2[1] = 0, q2[0] = two(s.s1, 0.f), q2[1] = 0;
    }
    __device__ __forceinline__ void add(uint64_t x, int i) {
        float e0, e1;
        const uint64_t d = add_two(x, minus);
        apart(mul_two(d, two(c, c)), e0, e1);
        const uint64_t e = two(exp2_fast(e0), exp2_fast(e1));
        t2[i] = add_two(t2[i], e);
        if (MODE == kSquare) q2[i] = fma_two(e, e, q2[i]);
        if (MODE == kBoth) {
            apart(mul_two(d, two(kLog2e, kLog2e)), e0, e1);
            q2[i] = add_two(q2[i], two(exp2_fast(e0), exp2_fast(e1)));
        }
    }
    __device__ __forceinline__ void take(float x) {
        if (x > limit) move_to(x);
        add(two(x, -INFINITY), 0);
    }
    template <typename T, int U> __device__ __forceinline__ void take(const uint4 (&u)[U]) {
        const float top = top_of(u, T());
        if (top > limit) move_to(top);
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const Pairs<T> p(u[k]);
#pragma unroll
            for (int i = 0; i < Pairs<T>::count; ++i) add(p.x[i], i & 1);
        }
    }
};

// the part [lo, hi) of a row of `n` elements that block `r` of `blocks` takes;
// boundaries on 16-byte addresses, `head` elements before the first of them
__device__ __forceinline__ void part_of(int64_t n, int64_t head, int per16, int r, int blocks, int64_t &lo, int64_t &hi) {
    const int64_t body = n > head ? (n - head + per16 - 1) / per16 : 0;
    const int64_t per = (body + blocks - 1) / blocks;
    lo = r == 0 ? 0 : min(n, head + r * per * per16);
    hi = r == blocks - 1 ? n : min(n, head + (r + 1) * per * per16);
}

// The teacher's side of a row, in one warp: softmax over its valid entries,
// and the divergence from the student's log probabilities.  The first entries
// and the student's logits there are loaded ahead.
struct Teacher {
    static constexpr int E = 4;
    int64_t ids[E];
    float t[E], x[E];
    __device__ __forceinline__ static bool valid(const Args &a, int64_t id) { return id >= 0 && id < a.V; }
    __device__ __forceinline__ void entries(const Args &a, int64_t row, int lane) {
#pragma unroll
        for (int k = 0; k < E; ++k) {
            const bool on = a.hard != 1.f && lane + 32 * k < a.K;
            ids[k] = on ? id_at(a, row * a.K + lane + 32 * k) : -1;
            t[k] = on ? teacher_at(a, row * a.K + lane + 32 * k) : 0.f;
        }
    }
    template <typename T> __device__ __forceinline__ void logits(const Args &a, const T *z) {
#pragma unroll
        for (int k = 0; k < E; ++k) x[k] = valid(a, ids[k]) ? to_f(z[ids[k]]) : 0.f;
    }
    // the row's loss and what backward needs of it, from the sums over the row
    template <typename T, int MODE>
    __device__ __forceinline__ void finish(const Args &a, int64_t row, const T *z, int lane, float m, float s1, float st, float zy) {
        const int64_t base = row * a.K;
        float tmax = -INFINITY, tsum = 0.f, kl = 0.f;
        bool any = false;  // an entry that counts; what is not finite among them makes the row NaN
        if (a.hard != 1.f) {
#pragma unroll
            for (int k = 0; k < E; ++k)
                if (valid(a, ids[k])) any = true, tmax = fmaxf(tmax, t[k]);
            for (int k = lane + 32 * E; k < a.K; k += 32)
                if (valid(a, id_at(a, base + k))) any = true, tmax = fmaxf(tmax, teacher_at(a, base + k));
            tmax = warp_max(tmax);
            any = __any_sync(0xffffffffu, any);
            if (any) {
#pragma unroll
                for (int k = 0; k < E; ++k)
                    if (valid(a, ids[k])) tsum += expf((t[k] - tmax) * a.inv_tau);
                for (int k = lane + 32 * E; k < a.K; k += 32)
                    if (valid(a, id_at(a, base + k))) tsum += expf((teacher_at(a, base + k) - tmax) * a.inv_tau);
                tsum = warp_sum(tsum);
                const float log_tsum = logf(tsum), log_st = logf(st), inv = 1.f / tsum;
                auto entry = [&](float te, float xe) {
                    const float lt = (te - tmax) * a.inv_tau, p = expf(lt) * inv;
                    // p = 0 adds nothing, whatever the student says
                    if (p != 0.f) kl += p * ((lt - log_tsum) - ((xe - m) * a.inv_tau - log_st));
                };
#pragma unroll
                for (int k = 0; k < E; ++k)
                    if (valid(a, ids[k])) entry(t[k], x[k]);
                for (int k = lane + 32 * E; k < a.K; k += 32) {
                    const int64_t id = id_at(a, base + k);
                    if (valid(a, id)) entry(teacher_at(a, base + k), to_f(z[id]));
                }
                kl = warp_sum(kl);
            }
        }
        if (lane != 0) return;
        float loss = 0.f;
        if (a.hard != 1.f) loss = (1.f - a.hard) * a.tau * a.tau * kl;
        // exp(z - m) summed: the one sum of kOne (tau = 1 or labels alone), s1 otherwise
        if (a.hard != 0.f) loss += a.hard * (logf(MODE == kOne ? st : s1) + (m - zy));
        a.rows[row] = loss;
        float *q = a.stats + row * kStats;
        q[0] = m;
        q[1] = MODE == kOne ? st : s1;
        q[2] = st;
        q[3] = tmax;
        q[4] = any ? 1.f / tsum : 0.f;
        q[5] = 1.f;
    }
};

template <typename T, int MODE>
__global__ void __launch_bounds__(kThreads) distill_kernel(const Args a) {
    constexpr int N = 16 / (int)sizeof(T);
    using V = Vec<T, N>;
    cg::cluster_group cl = cg::this_cluster();
    const int blocks = (int)cl.num_blocks(), r = (int)cl.block_rank();
    const int64_t row = blockIdx.x / blocks;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __shared__ float red[3][kWarps];
    __shared__ float part[3];
    // a row that is left out is not read
    const int64_t y = a.targets ? a.targets[row] : 0;
    const bool counts = y >= 0 && y < a.V;  // the same in every block of the cluster
    if (!counts) {
        if (r == 0 && tid == 0) a.rows[row] = 0.f, a.stats[row * kStats + 5] = 0.f;
        return;
    }
    const T *z = static_cast<const T *>(a.z) + row * a.ldz;
    const float c = (MODE == kOne && a.hard == 1.f ? 1.f : a.inv_tau) * kLog2e;

    // the first warp of the row's first block will need the teacher's entries:
    // the first of them are on their way from here
    Teacher teacher;
    if (r == 0 && warp == 0) teacher.entries(a, row, lane);
    const float zy = a.hard != 0.f && r == 0 && tid == 0 ? to_f(z[y]) : 0.f;

    Running<MODE> run(c);
    const int64_t head = min(a.V, (int64_t)((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / (int64_t)sizeof(T));
    int64_t lo, hi;
    part_of(a.V, head, N, r, blocks, lo, hi);
    if (r == 0) {
        for (int64_t i = tid; i < head; i += kThreads) run.take(to_f(z[i]));
        lo = head;
    }
    const int vecs = hi > lo ? (int)((hi - lo) / N) : 0;
    const uint4 *zv = reinterpret_cast<const uint4 *>(z + lo);
    constexpr int U = 4;  // vectors in flight per thread
    int i = tid;
    for (; i + (U - 1) * kThreads < vecs; i += U * kThreads) {
        uint4 x[U];
#pragma unroll
        for (int k = 0; k < U; ++k) x[k] = zv[i + k * kThreads];
        run.template take<T, U>(x);
    }
    for (; i < vecs; i += kThreads) {
        const uint4 x[1] = {zv[i]};
        run.template take<T, 1>(x);
    }
    if (r == 0 && warp == 0) teacher.logits(a, z);
    for (int64_t e = lo + (int64_t)vecs * N + tid; e < hi; e += kThreads) run.take(to_f(z[e]));
    Sums<MODE> s = run.sums();

#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, s.m, o), o1 = __shfl_xor_sync(0xffffffffu, s.s1, o),
                    ot = __shfl_xor_sync(0xffffffffu, s.st, o);
        s.join(om, o1, ot, c);
    }
    if (lane == 0) red[0][warp] = s.m, red[1][warp] = s.s1, red[2][warp] = s.st;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kWarps; ++w) s.join(red[0][w], red[1][w], red[2][w], c);
        part[0] = s.m, part[1] = s.s1, part[2] = s.st;
    }
    if (blocks > 1) {
        cl.sync();
        if (r == 0 && tid == 0)
            for (int b = 1; b < blocks; ++b) {
                const float *o = cl.map_shared_rank(part, b);
                s.join(o[0], o[1], o[2], c);
            }
        cl.sync();  // the other blocks stay until their sums are read
        if (r != 0) return;
        if (tid == 0) part[0] = s.m, part[1] = s.s1, part[2] = s.st;
    }
    __syncthreads();
    const float m = part[0], s1 = part[1], st = part[2];

    if (warp == 0) teacher.finish<T, MODE>(a, row, z, lane, m, s1, st, zy);
}

// loss = sum of the rows, or their mean over those that count, and the factor
// that this puts before every row.  One block, fixed order, 64 bits.
__global__ void __launch_bounds__(1024)
    distill_join_kernel(const float *rows, const float *stats, int64_t n, int mean, float *loss, float *factor) {
    __shared__ double sum[32];
    __shared__ double num[32];
    double s = 0, c = 0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) s += rows[i], c += stats[i * kStats + 5];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o), c += __shfl_xor_sync(0xffffffffu, c, o);
    if ((threadIdx.x & 31) == 0) sum[threadIdx.x >> 5] = s, num[threadIdx.x >> 5] = c;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 32; ++w) s += sum[w], c += num[w];
        const double f = mean ? (c > 0 ? 1.0 / c : 0.0) : 1.0;
        *loss = (float)(s * f);
        *factor = (float)f;
    }
}

// gradients without their teacher and label terms: at exp((z - m) / tau) + a1 exp(z - m)
template <int MODE> struct Smooth {
    float c, m, at, a1;
    __device__ __forceinline__ float one(float x) const {
        const float d = x - m, e = exp2_fast(d * c);
        if (MODE == kOne) return at * e;
        if (MODE == kSquare) return e * fmaf(a1, e, at);
        return fmaf(at, e, a1 * exp2_fast(d * kLog2e));
    }
    __device__ __forceinline__ uint64_t pair(uint64_t x) const {
        float e0, e1;
        const uint64_t d = add_two(x, two(-m, -m));
        apart(mul_two(d, two(c, c)), e0, e1);
        const uint64_t e = two(exp2_fast(e0), exp2_fast(e1)), t = two(at, at), q = two(a1, a1);
        if (MODE == kOne) return mul_two(t, e);
        if (MODE == kSquare) return mul_two(e, fma_two(q, e, t));
        apart(mul_two(d, two(kLog2e, kLog2e)), e0, e1);
        return fma_two(t, e, mul_two(q, two(exp2_fast(e0), exp2_fast(e1))));
    }
};
// 16 bytes of gradients from 16 bytes of logits
template <int MODE> __device__ __forceinline__ uint4 smooth16(const Smooth<MODE> &f, const uint4 &u, float) {
    const Pairs<float> p(u);
    float a, b, c, d;
    apart(f.pair(p.x[0]), a, b);
    apart(f.pair(p.x[1]), c, d);
    return make_uint4(__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d));
}
template <int MODE, typename T> __device__ __forceinline__ uint4 smooth16(const Smooth<MODE> &f, const uint4 &u, T t) {
    const Pairs<T> p(u);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a, b;
        apart(f.pair(p.x[i]), a, b);
        w[i] = pack2(a, b, t);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T, int MODE>
__global__ void __launch_bounds__(kThreads) distill_backward_kernel(const Args a, int blocks) {
    constexpr int N = 16 / (int)sizeof(T);
    using V = Vec<T, N>;
    __shared__ int32_t ids[CAIL_OPS_DISTILL_MAX_K + 1];
    __shared__ float terms[CAIL_OPS_DISTILL_MAX_K + 1];
    const int64_t row = blockIdx.x / blocks;
    const int r = (int)(blockIdx.x % blocks), tid = threadIdx.x;
    const T *z = static_cast<const T *>(a.z) + row * a.ldz;
    T *g = static_cast<T *>(a.grad) + row * a.ldg;
    const float *q = a.stats + row * kStats;
    const bool counts = q[5] != 0.f;
    // z and g rows on the same offset from a 16-byte address go by vectors
    const uintptr_t off = reinterpret_cast<uintptr_t>(g) & 15;
    const bool vec = off == (reinterpret_cast<uintptr_t>(z) & 15);
    const int64_t head = min(a.V, (int64_t)((16 - off) & 15) / (int64_t)sizeof(T));
    int64_t lo, hi;
    part_of(a.V, head, N, r, blocks, lo, hi);
    const int64_t from = lo;

    const float scale = counts ? a.grad_loss[a.per_row_grad ? row : 0] * (a.per_row_grad ? 1.f : *a.factor) : 0.f;
    if (!counts) {  // zeros, and the row is not read
        const T zero = from_f<T>(0.f);
        V zv;
#pragma unroll
        for (int k = 0; k < N; ++k) zv.v[k] = zero;
        if (r == 0) {
            for (int64_t i = tid; i < head; i += kThreads) g[i] = zero;
            lo = head;
        }
        const int64_t vecs = hi > lo ? (hi - lo) / N : 0;
        for (int64_t i = tid; i < vecs; i += kThreads) reinterpret_cast<V *>(g + lo)[i] = zv;
        for (int64_t e = lo + vecs * N + tid; e < hi; e += kThreads) g[e] = zero;
        return;
    }
    const float soft = (1.f - a.hard) * a.tau * scale;
    Smooth<MODE> f;
    f.c = (MODE == kOne && a.hard == 1.f ? 1.f : a.inv_tau) * kLog2e;
    f.m = base_of(q[0]);
    // the factors of exp((z - m) / tau) and of exp(z - m)
    f.at = q[4] != 0.f ? fmaf(0.f, q[4], soft / q[2]) : 0.f, f.a1 = a.hard * scale / q[1];
    if (MODE == kOne) f.at += f.a1;

    auto one = [&](int64_t i) { g[i] = from_f<T>(f.one(to_f(z[i]))); };
    if (vec) {
        if (r == 0) {
            for (int64_t i = tid; i < head; i += kThreads) one(i);
            lo = head;
        }
        const int vecs = hi > lo ? (int)((hi - lo) / N) : 0;
        const uint4 *zv = reinterpret_cast<const uint4 *>(z + lo);
        uint4 *gv = reinterpret_cast<uint4 *>(g + lo);
        constexpr int U = 2;
        int i = tid;
        for (; i + (U - 1) * kThreads < vecs; i += U * kThreads) {
            uint4 x[U];
#pragma unroll
            for (int k = 0; k < U; ++k) x[k] = zv[i + k * kThreads];
#pragma unroll
            for (int k = 0; k < U; ++k) gv[i + k * kThreads] = smooth16<MODE>(f, x[k], T());
        }
        for (; i < vecs; i += kThreads) gv[i] = smooth16<MODE>(f, zv[i], T());
        for (int64_t e = lo + (int64_t)vecs * N + tid; e < hi; e += kThreads) one(e);
    } else {
        for (int64_t e = lo + tid; e < hi; e += kThreads) one(e);
    }

    // the entries with a term of their own, those of this block's part: the
    // same id twice adds up, at its first place
    const int64_t base = row * a.K;
    const int K = q[4] != 0.f && soft != 0.f ? a.K : 0;
    for (int k = tid; k < K; k += kThreads) {
        const int64_t id = id_at(a, base + k);
        const bool here = id >= from && id < hi;
        ids[k] = here ? (int32_t)(id - from) : -1;
        terms[k] = here ? soft * expf((teacher_at(a, base + k) - q[3]) * a.inv_tau) * q[4] : 0.f;
    }
    int n = K;
    if (a.hard != 0.f) {
        if (tid == 0) {
            const int64_t y = a.targets[row];
            ids[n] = y >= from && y < hi ? (int32_t)(y - from) : -1;
            terms[n] = a.hard * scale;
        }
        ++n;
    }
    __syncthreads();  // also: the plain values of these entries are written
    for (int k = tid; k < n; k += kThreads) {
        const int32_t id = ids[k];
        if (id < 0) continue;
        bool first = true;
        for (int j = 0; j < k; ++j) first &= ids[j] != id;
        if (!first) continue;
        float t = terms[k];
        for (int j = k + 1; j < n; ++j)
            if (ids[j] == id) t += terms[j];
        const int64_t e = from + id;
        g[e] = from_f<T>(f.one(to_f(z[e])) - t);
    }
}

// ------------------------------------------------------------ many rows
//
// With rows for every SM, blocks stay and take row after row.  One thread
// streams the rows through a ring of shared memory with bulk copies (16 KB
// pieces, 64 KB a block, three blocks an SM), across the rows' ends, so the
// memory never waits for a row's reductions; 256 threads take the pieces from
// there.  Backward turns a piece into gradients in place, puts the teacher's
// and the label's terms in, and copies it out the same way.

constexpr int kMath = 256, kRingThreads = kMath + 32, kStages = 4, kPiece = 16384;

struct Ring {
    uint32_t data, full, free_;
    __device__ __forceinline__ void init(int readers) const {
        for (int s = 0; s < kStages; ++s) mbar_init(full + 8 * s, 1), mbar_init(free_ + 8 * s, readers);
        fence_barrier_init();
    }
};
// where the vectors of a row begin, and how many there are
template <typename T> struct RowShape {
    int64_t head;
    int64_t bytes;
    __device__ __forceinline__ RowShape(const T *z, int64_t V) {
        head = min(V, (int64_t)((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / (int64_t)sizeof(T));
        bytes = (V - head) * (int64_t)sizeof(T) / 16 * 16;
    }
    __device__ __forceinline__ int pieces() const { return (int)((bytes + kPiece - 1) / kPiece); }
};
__device__ __forceinline__ bool row_counts(const Args &a, int64_t row) {
    if (!a.targets) return true;
    const int64_t y = a.targets[row];
    return y >= 0 && y < a.V;
}
// the loading thread: every row of this block that counts, piece by piece
template <typename T> __device__ __forceinline__ void stream_rows(const Args &a, const Ring &ring, int *error) {
    uint32_t g = 0;
    for (int64_t row = blockIdx.x; row < a.N; row += gridDim.x) {
        if (!row_counts(a, row)) continue;
        const T *z = static_cast<const T *>(a.z) + row * a.ldz;
        const RowShape<T> shape(z, a.V);
        const char *src = reinterpret_cast<const char *>(z + shape.head);
        for (int64_t at = 0; at < shape.bytes; at += kPiece, ++g) {
            const uint32_t s = g % kStages;
            if (g >= kStages && !mbar_wait(ring.free_ + 8 * s, ((g / kStages) & 1) ^ 1)) {
                report(error);
                for (uint32_t k = g - kStages; k < g; ++k) mbar_wait(ring.full + 8 * (k % kStages), (k / kStages) & 1);
                return;
            }
            const uint32_t bytes = (uint32_t)min((int64_t)kPiece, shape.bytes - at);
            mbar_expect(ring.full + 8 * s, bytes);
            bulk_load(ring.data + s * kPiece, src + at, bytes, ring.full + 8 * s);
        }
    }
}
__device__ __forceinline__ void math_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t at) {
    uint4 u;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(at));
    return u;
}

// Forward: eight warps sum, one loads, and one has the teacher's side, so the
// chain of its loads and logarithms is not in the summing warps' way.  Bound by
// exponentials (62 % of their pipe) and issue (59 %): 8192 x 50257 bf16, tau 2,
// 823 MB in 155 us, 5.3 TB/s.  (Both passes took 657 us before the rings, 485
// with them, 430 since the exponentials are packed.)
template <typename T, int MODE>
__global__ void __launch_bounds__(kRingThreads + 32, 3) distill_ring_kernel(const Args a, int *error) {
    extern __shared__ __align__(128) char ring_raw[];
    __shared__ __align__(8) uint64_t bars[2 * kStages + 4];
    __shared__ float red[2][3][kMath / 32];  // the warps' sums of two rows
    const Ring ring = {smem_u32(ring_raw), smem_u32(bars), smem_u32(bars) + 8 * kStages};
    const uint32_t sums_full = ring.free_ + 8 * kStages, sums_free = sums_full + 16;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int s = 0; s < 2; ++s) mbar_init(sums_full + 8 * s, kMath / 32), mbar_init(sums_free + 8 * s, 1);
        ring.init(kMath / 32);
    }
    __syncthreads();
    if (warp == kMath / 32) {
        if (lane == 0) stream_rows<T>(a, ring, error);
        return;
    }
    const float c = (MODE == kOne && a.hard == 1.f ? 1.f : a.inv_tau) * kLog2e;
    uint32_t g = 0, done = 0;  // pieces and rows so far
    bool ok = true;
    int64_t y = a.targets ? a.targets[blockIdx.x] : 0;
    for (int64_t row = blockIdx.x; row < a.N; row += gridDim.x) {
        const bool counts = y >= 0 && y < a.V;
        const int64_t label = y;
        if (a.targets && row + gridDim.x < a.N) y = a.targets[row + gridDim.x];  // the next row's, ahead of its use
        const T *z = static_cast<const T *>(a.z) + row * a.ldz;
        const uint32_t set = done & 1, phase = (done >> 1) & 1;
        if (warp > kMath / 32) {  // the teacher's side
            if (!counts) {
                if (lane == 0) a.rows[row] = 0.f, a.stats[row * kStats + 5] = 0.f;
                continue;
            }
            Teacher teacher;
            teacher.entries(a, row, lane);
            const float zy = a.hard != 0.f ? to_f(z[label]) : 0.f;
            teacher.logits(a, z);
            ok = ok && mbar_wait(sums_full + 8 * set, phase);
            Sums<MODE> s;
            for (int w = 0; w < kMath / 32; ++w) s.join(red[set][0][w], red[set][1][w], red[set][2][w], c);
            __syncwarp();
            if (lane == 0) mbar_arrive(sums_free + 8 * set);
            teacher.finish<T, MODE>(a, row, z, lane, s.m, s.s1, s.st, zy);
            ++done;
            continue;
        }
        if (!counts) continue;
        const RowShape<T> shape(z, a.V);
        // elements before the first vector and behind the last: one for each of the last warp's threads
        const int64_t tail = shape.head + shape.bytes / (int64_t)sizeof(T), odd = shape.head + (a.V - tail);
        const int mine = tid - (kMath - 32);
        float loose = 0.f;
        if (mine >= 0 && mine < odd) loose = to_f(z[mine < shape.head ? mine : tail + mine - shape.head]);

        Running<MODE> run(c);
        for (int64_t at = 0; at < shape.bytes; at += kPiece, ++g) {
            const uint32_t st = g % kStages;
            ok = ok && mbar_wait(ring.full + 8 * st, (g / kStages) & 1);
            const int vecs = (int)(min((int64_t)kPiece, shape.bytes - at) / 16);
            const uint32_t src = ring.data + st * kPiece;
            if (vecs == kPiece / 16) {
                static_assert(kPiece / 16 == 4 * kMath);
                const uint4 u[4] = {lds16(src + tid * 16), lds16(src + (tid + kMath) * 16), lds16(src + (tid + 2 * kMath) * 16),
                                    lds16(src + (tid + 3 * kMath) * 16)};
                run.template take<T, 4>(u);
            } else {
                for (int i = tid; i < vecs; i += kMath) {
                    const uint4 u[1] = {lds16(src + i * 16)};
                    run.template take<T, 1>(u);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(ring.free_ + 8 * st);
        }
        if (mine >= 0 && mine < odd) run.take(loose);
        Sums<MODE> s = run.sums();
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const float om = __shfl_xor_sync(0xffffffffu, s.m, o), o1 = __shfl_xor_sync(0xffffffffu, s.s1, o),
                        ot = __shfl_xor_sync(0xffffffffu, s.st, o);
            s.join(om, o1, ot, c);
        }
        if (done >= 2) ok = ok && mbar_wait(sums_free + 8 * set, phase ^ 1);
        if (lane == 0) {
            red[set][0][warp] = s.m, red[set][1][warp] = s.s1, red[set][2][warp] = s.st;
            mbar_arrive(sums_full + 8 * set);
        }
        ++done;
    }
    if (!ok && lane == 0) report(error);
}

// Backward: a piece is turned into its gradients where it lies and stored from
// there by a bulk copy.  Bound by memory: 8192 x 50257 bf16, 1.65 GB in 269 us,
// 6.1 TB/s.
template <typename T, int MODE>
__global__ void __launch_bounds__(kRingThreads, 3) distill_backward_ring_kernel(const Args a, int *error) {
    constexpr int N = 16 / (int)sizeof(T);
    extern __shared__ __align__(128) char ring_raw[];
    __shared__ __align__(8) uint64_t bars[2 * kStages];
    __shared__ int32_t ids[CAIL_OPS_DISTILL_MAX_K + 1];
    __shared__ float terms[CAIL_OPS_DISTILL_MAX_K + 1];
    const Ring ring = {smem_u32(ring_raw), smem_u32(bars), smem_u32(bars) + 8 * kStages};
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) ring.init(1);
    __syncthreads();
    if (warp == kMath / 32) {
        if (lane == 0) stream_rows<T>(a, ring, error);
        return;
    }
    Smooth<MODE> f;
    f.c = (MODE == kOne && a.hard == 1.f ? 1.f : a.inv_tau) * kLog2e;
    const float factor = a.per_row_grad ? 1.f : a.grad_loss[0] * *a.factor;
    uint32_t g = 0;
    bool ok = true;
    for (int64_t row = blockIdx.x; row < a.N; row += gridDim.x) {
        T *out = static_cast<T *>(a.grad) + row * a.ldg;
        const T *z = static_cast<const T *>(a.z) + row * a.ldz;
        const RowShape<T> shape(z, a.V);
        const int64_t tail = shape.head + shape.bytes / (int64_t)sizeof(T), odd = shape.head + (a.V - tail);
        const int64_t loose = tid < odd ? (tid < shape.head ? tid : tail + tid - shape.head) : -1;
        if (!row_counts(a, row)) {  // zeros
            const T zero = from_f<T>(0.f);
            if (loose >= 0) out[loose] = zero;
            for (int64_t i = tid; i < shape.bytes / 16; i += kMath) reinterpret_cast<uint4 *>(out + shape.head)[i] = make_uint4(0, 0, 0, 0);
            continue;
        }
        const float *q = a.stats + row * kStats;
        const float scale = a.per_row_grad ? a.grad_loss[row] : factor;
        const float soft = (1.f - a.hard) * a.tau * scale;
        f.m = base_of(q[0]);
        f.at = q[4] != 0.f ? fmaf(0.f, q[4], soft / q[2]) : 0.f, f.a1 = a.hard * scale / q[1];
        if (MODE == kOne) f.at += f.a1;

        // the terms of single entries: the same id twice adds up, at its first place
        const int64_t base = row * a.K;
        const int K = q[4] != 0.f && soft != 0.f ? a.K : 0, n = K + (a.hard != 0.f ? 1 : 0);
        math_sync();  // the row before is done with them
        for (int k = tid; k < K; k += kMath) {
            const int64_t id = id_at(a, base + k);
            const bool on = id >= 0 && id < a.V;
            ids[k] = on ? (int32_t)id : -1;
            terms[k] = on ? soft * expf((teacher_at(a, base + k) - q[3]) * a.inv_tau) * q[4] : 0.f;
        }
        if (tid == 0 && n > K) ids[K] = (int32_t)a.targets[row], terms[K] = a.hard * scale;
        math_sync();
        int32_t own[4];  // what this thread puts in: up to 4 entries of its own (n <= 1025)
        float own_term[4];
        int owned = 0;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int k = tid + x * kMath;
            own[x] = -1;
            if (k >= n || ids[k] < 0) continue;
            bool first = true;
            for (int j = 0; j < k; ++j) first &= ids[j] != ids[k];
            if (!first) continue;
            float t = terms[k];
            for (int j = k + 1; j < n; ++j)
                if (ids[j] == ids[k]) t += terms[j];
            own[x] = ids[k], own_term[x] = t, owned = 1;
        }
        float rest = 0.f;  // the 1025th entry (a label beside 1024 teacher entries): thread 0's own
        int32_t rest_id = -1;
        if (tid == 0 && n > 4 * kMath) {
            rest_id = ids[n - 1], rest = terms[n - 1];
            for (int j = 0; j < n - 1; ++j)
                if (ids[j] == rest_id) rest_id = -1;  // added where it came first
        }

        int64_t at = 0;
        for (; at < shape.bytes; at += kPiece, ++g) {
            const uint32_t st = g % kStages;
            ok = ok && mbar_wait(ring.full + 8 * st, (g / kStages) & 1);
            const int bytes = (int)min((int64_t)kPiece, shape.bytes - at), vecs = bytes / 16;
            const uint32_t src = ring.data + st * kPiece;
            // this piece's entries: the logit is kept before the piece is overwritten
            const int64_t e0 = shape.head + at / (int64_t)sizeof(T), e1 = e0 + vecs * N;
            float keep[5];
#pragma unroll
            for (int x = 0; x < 4; ++x)
                if (owned && own[x] >= e0 && own[x] < e1) keep[x] = to_f(*reinterpret_cast<const T *>(ring_raw + st * kPiece + (own[x] - e0) * sizeof(T)));
            if (rest_id >= e0 && rest_id < e1) keep[4] = to_f(*reinterpret_cast<const T *>(ring_raw + st * kPiece + (rest_id - e0) * sizeof(T)));
            math_sync();
            for (int i = tid; i < vecs; i += kMath) {
                const uint4 y = smooth16<MODE>(f, lds16(src + i * 16), T());
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(src + i * 16), "r"(y.x), "r"(y.y), "r"(y.z), "r"(y.w) : "memory");
            }
            math_sync();
#pragma unroll
            for (int x = 0; x < 4; ++x)
                if (owned && own[x] >= e0 && own[x] < e1)
                    *reinterpret_cast<T *>(ring_raw + st * kPiece + (own[x] - e0) * sizeof(T)) = from_f<T>(f.one(keep[x]) - own_term[x]);
            if (rest_id >= e0 && rest_id < e1)
                *reinterpret_cast<T *>(ring_raw + st * kPiece + (rest_id - e0) * sizeof(T)) = from_f<T>(f.one(keep[4]) - rest);
            fence_async();
            math_sync();
            if (tid == 0) {
                bulk_store(reinterpret_cast<char *>(out + shape.head) + at, src, bytes);
                // the piece before has been read out by now, or soon is
                bulk_wait_read<1>();
                if (g > 0) mbar_arrive(ring.free_ + 8 * ((g - 1) % kStages));
            }
        }
        // the elements outside the vectors
        if (loose >= 0) {
            float t = 0.f;
            for (int j = 0; j < n; ++j)
                if (ids[j] == (int32_t)loose) t += terms[j];
            out[loose] = from_f<T>(f.one(to_f(z[loose])) - t);
        }
    }
    if (tid == 0) bulk_wait_all();
    if (!ok && lane == 0) report(error);
}

int check(const cail_ops_distill_args *d) {
    if (d->type < CAIL_OPS_F32 || d->type > CAIL_OPS_F16 || d->teacher_type < CAIL_OPS_F32 || d->teacher_type > CAIL_OPS_F16)
        return fail(CAIL_OPS_EINVAL, "distill: unknown element type");
    if (d->N < 0 || d->V < 1 || d->V > 0x7fffffff || d->ld_logits < 0 || d->K < 0 || d->K > CAIL_OPS_DISTILL_MAX_K)
        return fail(CAIL_OPS_EINVAL, "distill: bad sizes (N %lld V %lld K %d)", (long long)d->N, (long long)d->V, d->K);
    if (!(d->temperature > 0.f) || !(d->hard_weight >= 0.f && d->hard_weight <= 1.f) || (d->hard_weight > 0.f && !d->targets))
        return fail(CAIL_OPS_EINVAL, "distill: bad temperature or hard weight");
    return CAIL_OPS_OK;
}

Args args_of(const cail_ops_distill_args *d) {
    Args a = {};
    a.N = d->N, a.V = d->V, a.ldz = d->ld_logits, a.ldg = d->ld_grad;
    a.z = d->logits, a.grad = d->grad;
    a.ids = d->ids, a.teacher = d->teacher, a.targets = d->targets;
    a.grad_loss = d->grad_loss, a.factor = d->factor;
    a.rows = d->rows, a.stats = d->stats;
    a.K = d->K, a.ids64 = d->ids64, a.teacher_type = d->teacher_type, a.per_row_grad = d->mean == -1;
    a.inv_tau = 1.f / d->temperature, a.tau = d->temperature, a.hard = d->hard_weight;
    return a;
}

// (8192 x 50257 bf16, a label's weight between 0 and 1: tau 1, one sum, 148 us
// forward and 428 with the backward pass; tau 2, one exponential for two sums,
// 155 and 434; other tau, two exponentials, 240 and 567.)
int mode_of(const cail_ops_distill_args *d) {
    if (d->temperature == 1.f || d->hard_weight == 0.f || d->hard_weight == 1.f) return kOne;
    return d->temperature == 2.f ? kSquare : kBoth;
}

// blocks per row: as many as give every SM two blocks, at most 8 (a portable
// cluster), each with a vector for every thread or more
int blocks_per_row(int64_t N, int64_t V, size_t size, int sms) {
    int b = 1;
    while (b < 8 && N * b < 2 * (int64_t)sms && V * (int64_t)size / (b * 2) >= 16 * kThreads) b *= 2;
    return b;
}

// rows for every SM, of a piece or more
bool streams(const Args &a, size_t size) { return a.N >= sm_count() && a.V * (int64_t)size >= kPiece; }

template <typename T, int MODE> int launch(const Args &a, int blocks, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    launch_clusters(cfg, (unsigned)a.N, blocks, distill_kernel<T, MODE>, a);
    return launched("distill");
}
template <typename K> int ring(K kernel, int threads, const Args &a, const char *who, cudaStream_t st) {
    if (int rc = earlier_error(who)) return rc;
    int *error = device_error_flag();
    if (!error) return fail(CAIL_OPS_ECUDA, "%s: no error word for this device", who);
    constexpr int smem = kStages * kPiece;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return fail(CAIL_OPS_ECUDA, "%s: %s", who, cudaGetErrorString(e));
    const unsigned grid = (unsigned)min(a.N, 3 * (int64_t)sm_count());
    kernel<<<grid, threads, smem, st>>>(a, error);
    return launched(who);
}
template <typename T> int launch(const Args &a, int mode, int blocks, cudaStream_t st) {
    if (streams(a, sizeof(T))) {
        if (mode == kOne) return ring(distill_ring_kernel<T, kOne>, kRingThreads + 32, a, "distill", st);
        if (mode == kSquare) return ring(distill_ring_kernel<T, kSquare>, kRingThreads + 32, a, "distill", st);
        return ring(distill_ring_kernel<T, kBoth>, kRingThreads + 32, a, "distill", st);
    }
    if (mode == kOne) return launch<T, kOne>(a, blocks, st);
    if (mode == kSquare) return launch<T, kSquare>(a, blocks, st);
    return launch<T, kBoth>(a, blocks, st);
}
template <typename T> int launch_backward(const Args &a, int mode, int blocks, cudaStream_t st) {
    // in place in the ring: gradients must lie as the logits do, modulo 16 bytes
    if (streams(a, sizeof(T)) && ((uintptr_t)a.z - (uintptr_t)a.grad) % 16 == 0 && (a.ldz - a.ldg) * (int64_t)sizeof(T) % 16 == 0) {
        if (mode == kOne) return ring(distill_backward_ring_kernel<T, kOne>, kRingThreads, a, "distill backward", st);
        if (mode == kSquare) return ring(distill_backward_ring_kernel<T, kSquare>, kRingThreads, a, "distill backward", st);
        return ring(distill_backward_ring_kernel<T, kBoth>, kRingThreads, a, "distill backward", st);
    }
    const unsigned grid = (unsigned)(a.N * blocks);
    if (mode == kOne) distill_backward_kernel<T, kOne><<<grid, kThreads, 0, st>>>(a, blocks);
    else if (mode == kSquare) distill_backward_kernel<T, kSquare><<<grid, kThreads, 0, st>>>(a, blocks);
    else distill_backward_kernel<T, kBoth><<<grid, kThreads, 0, st>>>(a, blocks);
    return launched("distill backward");
}

}  // namespace
}  // namespace cailops

extern "C" int cail_ops_distill(const cail_ops_distill_args *d, cail_ops_stream stream) {
    using namespace cailops;
    if (int rc = check(d)) return rc;
    auto st = static_cast<cudaStream_t>(stream);
    if (d->N > 0) {
        const Args a = args_of(d);
        const int mode = mode_of(d), blocks = blocks_per_row(d->N, d->V, type_size(d->type), sm_count());
        if (d->N * blocks > 0x7fffffff) return fail(CAIL_OPS_EINVAL, "distill: too many rows");
        int rc = d->type == CAIL_OPS_F32    ? launch<float>(a, mode, blocks, st)
                 : d->type == CAIL_OPS_BF16 ? launch<__nv_bfloat16>(a, mode, blocks, st)
                                            : launch<__half>(a, mode, blocks, st);
        if (rc) return rc;
    }
    if (d->mean == -1) return CAIL_OPS_OK;
    distill_join_kernel<<<1, 1024, 0, st>>>(d->rows, d->stats, d->N, d->mean, d->loss, d->factor);
    return launched("distill join");
}

extern "C" int cail_ops_distill_backward(const cail_ops_distill_args *d, cail_ops_stream stream) {
    using namespace cailops;
    if (int rc = check(d)) return rc;
    if (d->N == 0) return CAIL_OPS_OK;
    auto st = static_cast<cudaStream_t>(stream);
    const Args a = args_of(d);
    const int mode = mode_of(d), blocks = blocks_per_row(d->N, d->V, type_size(d->type), sm_count());
    if (d->N * blocks > 0x7fffffff) return fail(CAIL_OPS_EINVAL, "distill: too many rows");
    return d->type == CAIL_OPS_F32    ? launch_backward<float>(a, mode, blocks, st)
           : d->type == CAIL_OPS_BF16 ? launch_backward<__nv_bfloat16>(a, mode, blocks, st)
                                      : launch_backward<__half>(a, mode, blocks, st);
}
