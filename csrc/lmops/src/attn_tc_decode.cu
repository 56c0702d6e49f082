// attn_tc_decode.cu — one token per sequence against a long 16-bit cache, on
// the tensor cores.
//
// The cache is the only large operand, so it takes the 128-row side of both
// products and up to 16 query heads that share a key head take the other:
//   S^T [128 keys x 16 heads] = K Q^T,   O^T [D x 16] += V^T P
// K and V tiles stream through shared memory by TMA and are never touched by
// a thread; 128 threads hold one key each, take 16 scores from tensor memory,
// agree on the heads' running maxima and put p into shared memory for the
// second product: in two parts of the cache's type, the second what rounding
// took from the first, in columns of their own, which the product has to spare
// (16 is its least; 32 for groups of more than 8, which have one buffer of p
// for two).  So o is off by its own rounding alone, and that costs nothing up
// to 8 heads a group (16 x 4096 keys, 8 heads of 128: 16.5 us either way) and
// 6 % beyond (8 x 16384 keys, 16 heads of 128: 32.9 us, 30.9 with p rounded).
// O^T stays in tensor memory and is rescaled only when a maximum has grown by
// more than 2^8; its halves are added at the end.
//
// The keys are the sinks (padded to 16) and then the window; they are split
// over the blocks of a cluster, which join over distributed shared memory.
// Bound by reading the cache: 2 blocks per SM with 96 KB of tiles in flight
// each.  64 sequences of up to 8192 tokens, 32 query and 8 key heads of 128,
// window 4096 and 16 sinks: 816 MB in 141 us, 5.8 TB/s; attn_decode.cu, whose
// threads multiply, took 647 us for it.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "attn.cuh"
#include "tc.cuh"

namespace cg = cooperative_groups;

namespace cailops {
namespace {

constexpr int kKeys = 128, kQueries = 16, kThreads = 192;  // kQueries: columns of the first product

// HEADS: query heads of a block, 8 or 16
template <int DP, int HEADS> struct Shape {
    static constexpr int panels = DP / 64;
    static constexpr int slots = DP == 64 ? 6 : 3;  // tiles of K and V in turn
    static constexpr int columns = 2 * HEADS, p_buffers = HEADS == 8 ? 2 : 1;
    static constexpr int tile_bytes = kKeys * DP * 2, q_bytes = kQueries * DP * 2, p_bytes = columns * kKeys * 2;
    static constexpr int smem = 1024 + slots * tile_bytes + q_bytes + p_buffers * p_bytes;
    static constexpr int barriers = 2 * slots + 2 + 2 + 3;
};

struct Maps {
    CUtensorMap k, v, k16, v16;  // boxes of 128 keys and of 16
};

__device__ __forceinline__ float warp_max_fast(float x) {
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T, int DP, int HEADS>
__global__ void __launch_bounds__(kThreads, 2) tc_decode_kernel(const AttnArgs a, const __grid_constant__ Maps maps) {
    using S = Shape<DP, HEADS>;
    constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ char raw[];
    __shared__ __align__(8) uint64_t bars[S::barriers];
    __shared__ uint32_t tmem_at;
    __shared__ float wmax[2][4][HEADS];
    __shared__ float bm[HEADS], bl[HEADS], wl[4][HEADS];
    const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
    const uint32_t st = base, sq = st + S::slots * S::tile_bytes, sp = sq + S::q_bytes;
    // [HEADS][DP], this block's sums: in the place of the tiles, when all of them are done with
    float *const bo = reinterpret_cast<float *>(raw + (base - smem_u32(raw)));
    const uint32_t bar0 = smem_u32(bars);
    const uint32_t full = bar0, free_ = full + 8 * S::slots, s_full = free_ + 8 * S::slots, p_full = s_full + 16, o_done = p_full + 16,
                   o_last = o_done + 8, q_full = o_last + 8;
    cg::cluster_group cl = cg::this_cluster();
    const int blocks = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int chunks = (a.group + HEADS - 1) / HEADS;
    const int b = blockIdx.z, hk = blockIdx.y / chunks, h0 = hk * a.group + (blockIdx.y % chunks) * HEADS;
    const int heads = min(HEADS, (hk + 1) * a.group - h0);
    const int tid = threadIdx.x, warp = warp_number(), lane = tid & 31;
    const int n = length_of(a, b);
    // the keys, numbered: the sinks before the window, up to a multiple of 16, then the window
    const int win0 = max(0, n - a.window), nsink = min(a.sinks, win0), pad = (nsink + 15) / 16 * 16, total = pad + n - win0;
    const int tiles = (total + kKeys - 1) / kKeys, per = (tiles + blocks - 1) / blocks;
    const int from = min(tiles, rank * per), count = min(tiles, from + per) - from;

    if (warp == 4) {
        tmem_alloc<64>(smem_u32(&tmem_at));
        if (lane == 0) tma_prefetch(&maps.k), tma_prefetch(&maps.v);
    }
    if (tid == 0) {
        for (int s = 0; s < S::slots; ++s) mbar_init(full + 8 * s, 1), mbar_init(free_ + 8 * s, 1);
        for (int s = 0; s < 2; ++s) mbar_init(s_full + 8 * s, 1), mbar_init(p_full + 8 * s, 4);
        mbar_init(o_done, 1), mbar_init(o_last, 1), mbar_init(q_full, 128);
        fence_barrier_init();
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tm = tmem_at;
    bool ok = true;

    if (count == 0) {
        if (tid < HEADS) bm[tid] = -INFINITY, bl[tid] = 0.f;
        for (int i = tid; i < HEADS * DP; i += kThreads) bo[i] = 0.f;
    } else if (warp == 4) {
        if (lane == 0) {  // loads
            int y = 0;
            for (; y < 2 * count; ++y) {
                const int s = y % S::slots, v0 = (from + y / 2) * kKeys;
                const bool is_v = y & 1;
                if (y >= S::slots) ok = mbar_wait(free_ + 8 * s, ((y / S::slots) & 1) ^ 1);
                if (!ok) break;
                const uint32_t bar = full + 8 * s, dst = st + s * S::tile_bytes;
                mbar_expect(bar, S::tile_bytes);
                for (int p = 0; p < S::panels; ++p) {
                    if (v0 >= pad || v0 + kKeys <= pad) {
                        tma_load(dst + p * kKeys * 128, is_v ? &maps.v : &maps.k, bar, p * 64, v0 >= pad ? win0 + v0 - pad : v0, hk, b);
                    } else {  // sinks and window in one tile
                        for (int g = 0; g < kKeys; g += 16)
                            tma_load(dst + p * kKeys * 128 + g * 128, is_v ? &maps.v16 : &maps.k16, bar, p * 64,
                                     v0 + g < pad ? v0 + g : win0 + v0 + g - pad, hk, b);
                    }
                }
            }
            if (!ok) {  // gave up: the copies in flight land before the block ends
                report(a.error);
                for (int z = max(0, y - S::slots); z < y; ++z) mbar_wait(full + 8 * (z % S::slots), (z / S::slots) & 1);
            }
        }
    } else if (warp == 5) {
        // products: the whole warp runs the loop, one lane issues
        const bool leader = elect_one();
        constexpr uint32_t kind_s = mma_kind<bf, kKeys, kQueries, false>();
        // A = V^T: its rows (D) run along the tile's rows: MN-major
        constexpr uint32_t kind_o = mma_kind<bf, 128, S::columns, false>() | (1u << 15);
        const int steps = (a.D + 15) / 16;
        // D = 64: rows 64 and up of the second product are not used; their operand lies 8 keys on, inside the tiles
        const uint64_t dt = operand(st, 0), dq = operand(sq, 0), dvt = operand(st, DP == 64 ? 1024 : kKeys * 128), dp = operand(sp, 0);
        auto scores = [&](int x) {
            const int y = 2 * x, s = y % S::slots;
            if (!warp_wait(full + 8 * s, (y / S::slots) & 1)) return false;
            tc_after();
            if (leader) {
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk)
                    if (kk < steps)
                        mma_ss(tm + (x & 1) * kQueries, moved(dt, s * S::tile_bytes + (kk / 4) * kKeys * 128 + (kk % 4) * 32),
                               moved(dq, (kk / 4) * kQueries * 128 + (kk % 4) * 32), kind_s, kk > 0);
                mma_commit(free_ + 8 * s);
                mma_commit(s_full + 8 * (x & 1));
            }
            __syncwarp();
            return true;
        };
        ok = warp_wait(q_full, 0) && scores(0) && (count < 2 || scores(1));
        for (int x = 0; x < count && ok; ++x) {
            const int y = 2 * x + 1, s = y % S::slots;
            ok = warp_wait(full + 8 * s, (y / S::slots) & 1) && warp_wait(p_full + 8 * (x & 1), (x >> 1) & 1);
            if (!ok) break;
            tc_after();
            if (leader) {
#pragma unroll
                for (int kk = 0; kk < kKeys / 16; ++kk)
                    mma_ss(tm + 2 * kQueries, moved(dvt, s * S::tile_bytes + kk * 2048),
                           moved(dp, x % S::p_buffers * S::p_bytes + (kk / 4) * S::columns * 128 + (kk % 4) * 32), kind_o, x > 0 || kk > 0);
                mma_commit(free_ + 8 * s);
                mma_commit(o_done);
            }
            __syncwarp();
            if (x + 2 < count) ok = scores(x + 2);
        }
        if (leader) {
            mma_commit(o_last);
            if (!ok) report(a.error);
        }
    } else {  // one key each
        // the queries, zeros beyond the heads and D, and zeros for p beyond the heads
        for (int i = tid; i < kQueries * DP / 8; i += 128) {
            const int g = i / (DP / 8), c = i % (DP / 8);
            uint4 x = make_uint4(0, 0, 0, 0);
            if (g < heads && c * 8 < a.D) x = *reinterpret_cast<const uint4 *>(a.q + b * a.qb + (h0 + g) * a.qh + c * 16);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(sq + (c / 8) * kQueries * 128 + g * 128 + (((c % 8) ^ (g & 7)) * 16)), "r"(x.x),
                         "r"(x.y), "r"(x.z), "r"(x.w)
                         : "memory");
        }
        for (int i = tid; i < S::p_buffers * S::p_bytes / 16; i += 128)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sp + i * 16), "r"(0) : "memory");
        fence_async();
        mbar_arrive(q_full);
        const uint32_t mine = tm + ((uint32_t)(warp * 32) << 16);
        float m[HEADS], l[HEADS];
#pragma unroll
        for (int g = 0; g < HEADS; ++g) m[g] = -INFINITY, l[g] = 0.f;
        for (int x = 0; x < count; ++x) {
            const int v = (from + x) * kKeys + tid;
            const bool valid = v < pad ? v < nsink : v < total;
            ok = ok && mbar_wait(s_full + 8 * (x & 1), (x >> 1) & 1);
            uint32_t u[16];
            float *f = reinterpret_cast<float *>(u);
            __syncwarp();
            tc_after();
            tc_ld16(mine + (x & 1) * kQueries, u);
            tc_wait_ld16(u);
#pragma unroll
            for (int g = 0; g < HEADS; ++g) {
                if (g >= heads) break;
                f[g] = valid ? f[g] * a.scale_log2 : -INFINITY;
                const float w = warp_max_fast(f[g]);
                if (lane == 0) wmax[x & 1][warp][g] = w;
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            bool turned = false;
            float turn[HEADS];
#pragma unroll
            for (int g = 0; g < HEADS; ++g) {
                turn[g] = 1.f;
                if (g >= heads) break;
                const float top = fmaxf(fmaxf(wmax[x & 1][0][g], wmax[x & 1][1][g]), fmaxf(wmax[x & 1][2][g], wmax[x & 1][3][g]));
                if (m[g] == -INFINITY) {
                    m[g] = top;  // nothing of this head is in O yet
                } else if (top - m[g] > 8.f) {
                    turn[g] = exp2_fast(m[g] - top);
                    l[g] *= turn[g];
                    m[g] = top;
                    turned = true;
                }
            }
            // `turned` is the same in all 128 threads; with one buffer of p the product before has to be done with it
            if (turned || (S::p_buffers == 1 && x > 0)) {
                ok = ok && mbar_wait(o_done, (x - 1) & 1);
                __syncwarp();
                tc_after();
            }
            if (turned) {
                uint32_t w[S::columns];
                tc_ld<S::columns>(mine + 2 * kQueries, w);
                tc_wait_n<S::columns>(w);
#pragma unroll
                for (int g = 0; g < S::columns; ++g) w[g] = __float_as_uint(__uint_as_float(w[g]) * turn[g % HEADS]);
                if constexpr (S::columns == 16) tc_st16(mine + 2 * kQueries, w);
                else tc_st32(mine + 2 * kQueries, w);
                tc_wait_st();
            }
            const uint32_t col = sp + x % S::p_buffers * S::p_bytes + (tid / 64) * S::columns * 128 + (tid % 8) * 2;
#pragma unroll
            for (int g = 0; g < HEADS; ++g) {
                if (g >= heads) break;
                const float p = exp2_fast(f[g] - (m[g] == -INFINITY ? 0.f : m[g]));
                l[g] += p;
                const T t[2] = {from_f<T>(p), from_f<T>(rest_of<T>(p))};
#pragma unroll
                for (int part = 0; part < 2; ++part)
                    asm volatile("st.shared.b16 [%0], %1;" ::"r"(col + (part * HEADS + g) * 128 + (((tid % 64) / 8) ^ (g & 7)) * 16),
                                 "h"(*reinterpret_cast<const uint16_t *>(&t[part]))
                                 : "memory");
            }
            if (!valid) {  // what a key that is not seen holds may be infinite: its values are zeroed
                const int y = 2 * x + 1, s = y % S::slots;
                ok = ok && mbar_wait(full + 8 * s, (y / S::slots) & 1);
#pragma unroll
                for (int c = 0; c < DP / 8; ++c)
                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(st + s * S::tile_bytes + (c / 8) * kKeys * 128 + tid * 128 + (c % 8) * 16),
                                 "r"(0)
                                 : "memory");
            }
            __syncwarp();
            fence_async();
            tc_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * (x & 1));
        }
        ok = ok && mbar_wait(o_last, 0);
        __syncwarp();
        if (!ok && lane == 0) report(a.error);
        tc_after();
        uint32_t w[S::columns];
        tc_ld<S::columns>(mine + 2 * kQueries, w);
        tc_wait_n<S::columns>(w);
        if (tid < DP)
#pragma unroll
            for (int g = 0; g < HEADS; ++g) bo[g * DP + tid] = __uint_as_float(w[g]) + __uint_as_float(w[HEADS + g]);
#pragma unroll
        for (int g = 0; g < HEADS; ++g) {
            if (g >= heads) break;
            const float sum = warp_sum(l[g]);
            if (lane == 0) wl[warp][g] = sum;
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (tid < heads) bl[tid] = (wl[0][tid] + wl[1][tid]) + (wl[2][tid] + wl[3][tid]);
#pragma unroll
        for (int g = 0; g < HEADS; ++g)
            if (tid == g) bm[g] = m[g];
        tc_before();
    }
    __syncwarp();
    cl.sync();
    // blocks of the cluster: each joins a part of the output
    for (int i = rank * kThreads + tid; i < heads * a.D; i += blocks * kThreads) {
        const int g = i / a.D, d = i % a.D;
        float top = -INFINITY;
        for (int r = 0; r < blocks; ++r) top = fmaxf(top, *cl.map_shared_rank(&bm[g], r));
        const float off = top == -INFINITY ? 0.f : top;
        float x = 0.f, sum = 0.f;
        for (int r = 0; r < blocks; ++r) {
            const float f = exp2_fast(*cl.map_shared_rank(&bm[g], r) - off);
            x = fmaf(*cl.map_shared_rank(bo + g * DP + d, r), f, x);
            sum = fmaf(*cl.map_shared_rank(&bl[g], r), f, sum);
        }
        reinterpret_cast<T *>(a.o + b * a.ob + (h0 + g) * a.oh)[d] = from_f<T>(sum == 0.f ? 0.f : x / sum);
    }
    cl.sync();  // the others' sums stay until they are read
    if (warp == 4) tmem_free<64>(tm);
}

template <typename T, int DP, int HEADS> int launch(const cail_ops_attention_args *c, const AttnArgs &a, cudaStream_t st) {
    using S = Shape<DP, HEADS>;
    Maps maps;
    if (int rc = tensor_map(&maps.k, c->k, c->type, a.B, a.T, a.Hkv, a.D, kKeys)) return rc;
    if (int rc = tensor_map(&maps.v, c->v, c->type, a.B, a.T, a.Hkv, a.D, kKeys)) return rc;
    if (int rc = tensor_map(&maps.k16, c->k, c->type, a.B, a.T, a.Hkv, a.D, 16)) return rc;
    if (int rc = tensor_map(&maps.v16, c->v, c->type, a.B, a.T, a.Hkv, a.D, 16)) return rc;
    cudaError_t e = cudaFuncSetAttribute(tc_decode_kernel<T, DP, HEADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem);
    if (e != cudaSuccess) return fail(CAIL_OPS_ECUDA, "window attention decode: %s", cudaGetErrorString(e));
    e = cudaFuncSetAttribute(tc_decode_kernel<T, DP, HEADS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return fail(CAIL_OPS_ECUDA, "window attention decode: %s", cudaGetErrorString(e));
    const int chunks = (a.group + HEADS - 1) / HEADS;
    const int64_t work = (int64_t)a.B * a.Hkv * chunks, keys = std::min((int64_t)a.T, (int64_t)a.window + a.sinks);
    // Blocks per sequence and group: as many as give every SM up to two, each
    // with two tiles or more.  More of them only add their starts and joins
    // (64 sequences x 8 groups of 4096 keys, D 128: 170 us with 1, 185 with 2,
    // 206 with 4).  Clusters of 16 only while they get an SM each: 8 groups of
    // 16384 keys, 19.5 us against 29.6 with 8; 16 groups, 44 against 40.
    const int64_t sms = sm_count();
    int blocks = 1;
    while (blocks < 16 && work * blocks * 2 <= (blocks < 8 ? 2 * sms : sms) && keys >= blocks * 2 * 2 * kKeys) blocks *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1, a.Hkv * chunks, a.B);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = S::smem;
    cfg.stream = st;
    launch_clusters(cfg, 1, blocks, tc_decode_kernel<T, DP, HEADS>, a, maps);
    return launched("window attention decode");
}

template <typename T> int sized(const cail_ops_attention_args *c, const AttnArgs &a, cudaStream_t st) {
    if (a.group <= 8) return a.D <= 64 ? launch<T, 64, 8>(c, a, st) : launch<T, 128, 8>(c, a, st);
    return a.D <= 64 ? launch<T, 64, 16>(c, a, st) : launch<T, 128, 16>(c, a, st);
}

}  // namespace

// 16-bit caches in rows that TMA can load, and enough of them: below this the
// other kernel's shorter start wins (one head of 64: 256 keys 5.0 against
// 7.3 us, 1024 keys 6.9 against 7.5, 4096 keys 16 against 10; a group of four
// heads of 128: 64 keys 10.5 against 9.3, 1024 keys 15 against 9.3)
bool tc_takes_decode(const cail_ops_attention_args *a) {
    if (a->type == CAIL_OPS_F32 || a->D % 8 || a->T < 1) return false;
    if (!rows_aligned(a->q, a->B, 1, a->H, 2, 16) || !tma_takes(a->k, a->B, a->T, a->Hkv) || !tma_takes(a->v, a->B, a->T, a->Hkv)) return false;
    const int64_t keys = std::min((int64_t)a->T, (int64_t)a->window + a->sinks);
    return keys * (a->H / a->Hkv >= 4 ? 2 : 1) * (a->D > 64 ? 2 : 1) >= 1024;
}

int tc_decode(const cail_ops_attention_args *c, cudaStream_t st) {
    AttnArgs a = attn_args(c, false);
    if (int rc = earlier_error("window attention decode")) return rc;
    a.error = device_error_flag();
    if (!a.error) return fail(CAIL_OPS_ECUDA, "window attention decode: no error word for this device");
    return c->type == CAIL_OPS_BF16 ? sized<__nv_bfloat16>(c, a, st) : sized<__half>(c, a, st);
}

}  // namespace cailops
