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
#include <cooperative_groups.h>

#include "ops_common.cuh"

namespace cg = cooperative_groups;

namespace cailops {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;

// what forward keeps of a row: [0] m, [1] sum exp(z - m), [2] sum exp((z - m) / tau),
// [3] the teacher's maximum of t / tau, [4] 1 / sum exp(t / tau - max) (0: no teacher entry), [5] 1 if the row counts
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

// MODE of the sums: which of exp(z - m) and exp((z - m) / tau) are needed.
// kSquare: both with tau = 2, where the first is the second squared.
enum { kOne, kSquare, kBoth };

template <int MODE> struct Sums {
    float m = -INFINITY, s1 = 0.f, st = 0.f;
    // kOne keeps one sum, st, at the scale `c` (1 / tau, or 1 for the label alone)
    __device__ __forceinline__ static float base(float m) { return m == -INFINITY ? 0.f : m; }
    __device__ __forceinline__ void scale_to(float n, float c) {
        if (n == m) return;
        const float d = base(m) - base(n);  // m = -inf: sums are 0
        if (MODE == kOne) st *= exp2_fast(d * c);
        if (MODE == kSquare) {
            const float e = exp2_fast(d * c);
            st *= e, s1 *= e * e;
        }
        if (MODE == kBoth) st *= exp2_fast(d * c), s1 *= exp2_fast(d * kLog2e);
        m = n;
    }
    __device__ __forceinline__ void add(float x, float b, float c) {
        const float e = exp2_fast((x - b) * c);
        st += e;
        if (MODE == kSquare) s1 = fmaf(e, e, s1);
        if (MODE == kBoth) s1 += exp2_fast((x - b) * kLog2e);
    }
    template <int N> __device__ __forceinline__ void take(const float *x, float c) {
        float n = m;
#pragma unroll
        for (int i = 0; i < N; ++i) n = fmaxf(n, x[i]);
        scale_to(n, c);
        const float b = base(m);
#pragma unroll
        for (int i = 0; i < N; ++i) add(x[i], b, c);
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

// the part [lo, hi) of a row of `n` elements that block `r` of `blocks` takes;
// boundaries on 16-byte addresses, `head` elements before the first of them
__device__ __forceinline__ void part_of(int64_t n, int64_t head, int per16, int r, int blocks, int64_t &lo, int64_t &hi) {
    const int64_t body = n > head ? (n - head + per16 - 1) / per16 : 0;
    const int64_t per = (body + blocks - 1) / blocks;
    lo = r == 0 ? 0 : min(n, head + r * per * per16);
    hi = r == blocks - 1 ? n : min(n, head + (r + 1) * per * per16);
}

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

    Sums<MODE> s;
    const int64_t head = min(a.V, (int64_t)((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / (int64_t)sizeof(T));
    int64_t lo, hi;
    part_of(a.V, head, N, r, blocks, lo, hi);
    if (r == 0) {
        for (int64_t i = tid; i < head; i += kThreads) {
            const float x = to_f(z[i]);
            s.template take<1>(&x, c);
        }
        lo = head;
    }
    const int64_t vecs = hi > lo ? (hi - lo) / N : 0;
    const V *zv = reinterpret_cast<const V *>(z + lo);
    constexpr int U = 4;  // vectors in flight per thread
    int64_t i = tid;
    for (; i + (U - 1) * kThreads < vecs; i += U * kThreads) {
        V x[U];
#pragma unroll
        for (int k = 0; k < U; ++k) x[k] = zv[i + k * kThreads];
        float f[U * N];
#pragma unroll
        for (int k = 0; k < U * N; ++k) f[k] = to_f(x[k / N].v[k % N]);
        s.template take<U * N>(f, c);
    }
    for (; i < vecs; i += kThreads) {
        const V x = zv[i];
        float f[N];
#pragma unroll
        for (int k = 0; k < N; ++k) f[k] = to_f(x.v[k]);
        s.template take<N>(f, c);
    }
    for (int64_t e = lo + vecs * N + tid; e < hi; e += kThreads) {
        const float x = to_f(z[e]);
        s.template take<1>(&x, c);
    }

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

    // the teacher's side, one warp: softmax over its valid entries, then the
    // divergence from the student's log probabilities
    if (warp != 0) return;
    const int64_t base = row * a.K;
    float tmax = -INFINITY, tsum = 0.f, kl = 0.f;
    if (a.hard != 1.f) {
        for (int k = lane; k < a.K; k += 32) {
            const int64_t id = id_at(a, base + k);
            if (id >= 0 && id < a.V) tmax = fmaxf(tmax, teacher_at(a, base + k) * a.inv_tau);
        }
        tmax = warp_max(tmax);
        if (tmax != -INFINITY) {
            for (int k = lane; k < a.K; k += 32) {
                const int64_t id = id_at(a, base + k);
                if (id >= 0 && id < a.V) tsum += expf(teacher_at(a, base + k) * a.inv_tau - tmax);
            }
            tsum = warp_sum(tsum);
            const float log_tsum = logf(tsum), log_st = logf(st), inv = 1.f / tsum;
            for (int k = lane; k < a.K; k += 32) {
                const int64_t id = id_at(a, base + k);
                if (id < 0 || id >= a.V) continue;
                const float lt = teacher_at(a, base + k) * a.inv_tau - tmax;
                const float p = expf(lt) * inv;
                // p = 0 adds nothing, whatever the student says
                if (p > 0.f) kl += p * ((lt - log_tsum) - ((to_f(z[id]) - m) * a.inv_tau - log_st));
            }
            kl = warp_sum(kl);
        }
    }
    if (lane == 0) {
        float loss = 0.f;
        if (a.hard != 1.f) loss = (1.f - a.hard) * a.tau * a.tau * kl;
        if (a.hard != 0.f) {
            // exp(z - m) summed: the one sum of kOne (tau = 1 or labels alone), s1 otherwise
            loss += a.hard * (logf(MODE == kOne ? st : s1) + (m - to_f(z[y])));
        }
        a.rows[row] = loss;
        float *q = a.stats + row * kStats;
        q[0] = m;
        q[1] = MODE == kOne ? st : s1;
        q[2] = st;
        q[3] = tmax;
        q[4] = tmax == -INFINITY ? 0.f : 1.f / tsum;
        q[5] = 1.f;
    }
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

// one element's gradient without its teacher and label terms
template <int MODE>
__device__ __forceinline__ float smooth(float x, float m, float c, float at, float a1) {
    const float e = exp2_fast((x - m) * c);
    if (MODE == kOne) return at * e;
    if (MODE == kSquare) return e * fmaf(a1, e, at);
    return fmaf(at, e, a1 * exp2_fast((x - m) * kLog2e));
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
    const float m = q[0] == -INFINITY ? 0.f : q[0];
    const float c = (MODE == kOne && a.hard == 1.f ? 1.f : a.inv_tau) * kLog2e;
    const float soft = (1.f - a.hard) * a.tau * scale;
    // the factors of exp((z - m) / tau) and of exp(z - m)
    float at = q[4] != 0.f ? soft / q[2] : 0.f, a1 = a.hard * scale / q[1];
    if (MODE == kOne) at += a1;

    auto one = [&](int64_t i) { g[i] = from_f<T>(smooth<MODE>(to_f(z[i]), m, c, at, a1)); };
    if (vec) {
        if (r == 0) {
            for (int64_t i = tid; i < head; i += kThreads) one(i);
            lo = head;
        }
        const int64_t vecs = hi > lo ? (hi - lo) / N : 0;
        const V *zv = reinterpret_cast<const V *>(z + lo);
        V *gv = reinterpret_cast<V *>(g + lo);
        constexpr int U = 2;
        int64_t i = tid;
        for (; i + (U - 1) * kThreads < vecs; i += U * kThreads) {
            V x[U];
#pragma unroll
            for (int k = 0; k < U; ++k) x[k] = zv[i + k * kThreads];
#pragma unroll
            for (int k = 0; k < U; ++k) {
#pragma unroll
                for (int j = 0; j < N; ++j) x[k].v[j] = from_f<T>(smooth<MODE>(to_f(x[k].v[j]), m, c, at, a1));
                gv[i + k * kThreads] = x[k];
            }
        }
        for (; i < vecs; i += kThreads) {
            V x = zv[i];
#pragma unroll
            for (int j = 0; j < N; ++j) x.v[j] = from_f<T>(smooth<MODE>(to_f(x.v[j]), m, c, at, a1));
            gv[i] = x;
        }
        for (int64_t e = lo + vecs * N + tid; e < hi; e += kThreads) one(e);
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
        terms[k] = here ? soft * expf(teacher_at(a, base + k) * a.inv_tau - q[3]) * q[4] : 0.f;
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
        g[e] = from_f<T>(smooth<MODE>(to_f(z[e]), m, c, at, a1) - t);
    }
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

template <typename T, int MODE> int launch(const Args &a, int blocks, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.N * blocks));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)blocks, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, distill_kernel<T, MODE>, a);
    return launched("distill");
}
template <typename T> int launch(const Args &a, int mode, int blocks, cudaStream_t st) {
    if (mode == kOne) return launch<T, kOne>(a, blocks, st);
    if (mode == kSquare) return launch<T, kSquare>(a, blocks, st);
    return launch<T, kBoth>(a, blocks, st);
}
template <typename T> int launch_backward(const Args &a, int mode, int blocks, cudaStream_t st) {
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
