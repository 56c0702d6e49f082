// attn_tc_forward.cu — window attention on the tensor cores (bf16, fp16).
//
// A block owns 128 query rows of one head and goes once over the key tiles
// (64 keys) that some of them see.  One thread loads tiles by TMA, one issues
// the matrix products, 128 threads hold one row each: S = Q K^T arrives in
// tensor memory (two buffers, so the next product runs under this softmax),
// the row's thread keeps the running maximum and sum in registers without any
// exchange, writes p back over S as 16-bit, and O += P V takes it from there.
// O stays in tensor memory; it is rescaled only when a row's maximum has grown
// by more than 2^8 since the scale in use, so p stays below 256 and most tiles
// touch O in no other way than the product.  p is rounded to the input type
// for that product (its sum is not), as a second part of it would double the
// product, 40 % more for the tensor pipe; everything else is 32-bit.  Rows of few
// keys (cail_ops_rest_rows) take p in two parts, the second what rounding took
// from the first, and so twice the second product, in loops of their own (one
// loop with the choice inside took 3 % more): 0.4 us of 34 below.
//
// 64 keys per tile, two blocks per SM with two buffers of S each, so a product
// runs under the softmax.  4 x 4096 tokens, 16 heads, causal: 217 us at D = 64,
// 280 at D = 128, 635 and 980 TFLOP/s, about 900 and 1160 clocks a tile and SM.
// A tile's exponentials take 512 of them (16 a clock and SM), its products 334
// at D = 64 and 664 at D = 128 (50 for a 64-column product from shared memory,
// whose operations alone are 32, and 33 from tensor memory).  So at D = 64
// neither bounds it by itself, as a quarter of the exponentials on the float
// pipes, which measured the same, says too: the softmax warps wait on their own
// row's chain (scores out, maximum, exponentials, p back).
// Four blocks per SM with one buffer each measured the same; small calls took
// 8 us instead of 6.
//
// Short windows are bound by neither: 8 x 1024 tokens, 16 heads of 64, window
// 256 and 4 sinks, take 34 us (products 15 % of the tensor pipe, exponentials
// 35 %), as a block has five tiles between its prologue and its epilogue.
#include <type_traits>

#include "attn.cuh"
#include "tc.cuh"

namespace cailops {
namespace {

constexpr int kRows = 128, kKeys = 64, kThreads = 192;

template <int DP> struct Shape {
    static constexpr int panels = DP / 64;
    static constexpr int stages = DP == 64 ? 4 : 2;
    static constexpr int buffers = 2;  // of S
    static constexpr int per_sm = 2, columns = 256;
    static constexpr int q_bytes = kRows * DP * 2, kv_bytes = kKeys * DP * 2;
    static constexpr int barriers = 1 + 4 * stages + 2 + 2 + 2;
    static constexpr int smem = 1024 + q_bytes + 2 * stages * kv_bytes;
    static constexpr int o_col = buffers * kKeys;  // S, O
};

struct Maps {
    CUtensorMap q, k, v;
};

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, Shape<DP>::per_sm) tc_forward_kernel(const AttnArgs a, const __grid_constant__ Maps maps) {
    using S = Shape<DP>;
    constexpr int NB = S::buffers;
    constexpr bool bf = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ char raw[];
    __shared__ __align__(8) uint64_t bars[S::barriers];
    __shared__ uint32_t tmem_at;
    const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
    const uint32_t sq = base, sk = sq + S::q_bytes, sv = sk + S::stages * S::kv_bytes;
    const uint32_t bar0 = smem_u32(bars);
    auto bar = [&](int i) { return bar0 + 8u * i; };
    const uint32_t q_full = bar(0), k_full = bar(1), k_free = bar(1 + S::stages), v_full = bar(1 + 2 * S::stages),
                   v_free = bar(1 + 3 * S::stages), s_full = bar(1 + 4 * S::stages), p_full = s_full + 16, o_done = p_full + 16, o_last = o_done + 8;

    const int h = blockIdx.x, b = blockIdx.y, hk = h / a.group;
    const int i0 = (gridDim.z - 1 - blockIdx.z) * kRows;  // the longest rows first
    const int tid = threadIdx.x, warp = warp_number(), lane = tid & 31;
    const int n = length_of(a, b);
    const KeyTiles tiles(i0, i0 + kRows, n, a.window, a.sinks, kKeys);

    const bool fine = i0 < a.fine_rows;  // p in two parts

    if (tiles.count == 0) {  // rows behind the sequence: zeros
        constexpr int C = DP / 8;
        for (int i = tid; i < kRows * C; i += kThreads) {
            const int r = i0 + i / C, d = (i % C) * 8;
            if (r >= a.T || d >= a.D) continue;
            *reinterpret_cast<uint4 *>(a.o + b * a.ob + (int64_t)r * a.ot + h * a.oh + d * 2) = make_uint4(0, 0, 0, 0);
            if (r < a.rest_rows) *reinterpret_cast<uint4 *>(a.rest + b * a.rb + (int64_t)r * a.rt + h * a.rh + d * 2) = make_uint4(0, 0, 0, 0);
        }
        if (a.lse && tid < kRows && i0 + tid < a.T) a.lse[((int64_t)b * a.H + h) * a.lse_row + i0 + tid] = 0.f;
        return;
    }
    auto load_k = [&](int x) {
        const int s = x % S::stages, j0 = tiles.at(x) * kKeys;
        mbar_expect(k_full + 8 * s, S::kv_bytes);
        for (int p = 0; p < S::panels; ++p) tma_load(sk + s * S::kv_bytes + p * kKeys * 128, &maps.k, k_full + 8 * s, p * 64, j0, hk, b);
    };
    auto load_v = [&](int x) {
        const int s = x % S::stages, j0 = tiles.at(x) * kKeys;
        mbar_expect(v_full + 8 * s, S::kv_bytes);
        for (int p = 0; p < S::panels; ++p) tma_load(sv + s * S::kv_bytes + p * kKeys * 128, &maps.v, v_full + 8 * s, p * 64, j0, hk, b);
    };
    if (warp == 4 && lane == 0) {
        mbar_init(q_full, 1);
        for (int s = 0; s < S::stages; ++s) {
            mbar_init(k_full + 8 * s, 1), mbar_init(k_free + 8 * s, 1);
            mbar_init(v_full + 8 * s, 1), mbar_init(v_free + 8 * s, 1);
        }
        for (int s = 0; s < 2; ++s) mbar_init(s_full + 8 * s, 1), mbar_init(p_full + 8 * s, 4);
        mbar_init(o_done, 1), mbar_init(o_last, 1);
        fence_barrier_init();
        // what needs no free slot is on its way before the block has met
        mbar_expect(q_full, S::q_bytes);
        for (int p = 0; p < S::panels; ++p) tma_load(sq + p * kRows * 128, &maps.q, q_full, p * 64, i0, h, b);
        for (int x = 0; x < S::stages && x < tiles.count; ++x) load_k(x), load_v(x);
    }
    if (warp == 5) tmem_alloc<S::columns>(smem_u32(&tmem_at));
    __syncwarp();
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tm = tmem_at;
    bool ok = true;

    if (warp == 4) {
        if (lane == 0) {  // the loads that wait for a slot
            int x = S::stages;
            for (; x < tiles.count; ++x) {
                const int s = x % S::stages;
                const uint32_t before = ((x / S::stages) & 1) ^ 1;
                ok = mbar_wait(k_free + 8 * s, before);
                if (!ok) break;
                load_k(x);
                ok = mbar_wait(v_free + 8 * s, before);
                if (!ok) break;
                load_v(x);
            }
            if (!ok) {  // gave up: the copies in flight land before the block ends
                report(a.error);
                mbar_wait(q_full, 0);
                for (int y = x - S::stages; y < x; ++y)
                    mbar_wait(k_full + 8 * (y % S::stages), (y / S::stages) & 1), mbar_wait(v_full + 8 * (y % S::stages), (y / S::stages) & 1);
            }
        }
    } else if (warp == 5) {
        // products: the whole warp runs the loop, one lane issues
        const bool leader = elect_one();
        constexpr uint32_t kind_s = mma_kind<bf, kRows, kKeys, false>(), kind_o = mma_kind<bf, kRows, DP, true>();
        const int steps = (a.D + 15) / 16;
        const uint64_t dq = operand(sq, 0), dk = operand(sk, 0), dv = operand(sv, kKeys * 128);
        auto scores = [&](int x) {
            const int s = x % S::stages;
            if (!warp_wait(k_full + 8 * s, (x / S::stages) & 1)) return false;
            tc_after();
            const uint64_t dks = moved(dk, s * S::kv_bytes);
            const uint32_t d = tm + (x % NB) * kKeys;
            if (leader) {
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk)
                    if (kk < steps)
                        mma_ss(d, moved(dq, (kk / 4) * kRows * 128 + (kk % 4) * 32), moved(dks, (kk / 4) * kKeys * 128 + (kk % 4) * 32), kind_s,
                               kk > 0);
                mma_commit(k_free + 8 * s);
                mma_commit(s_full + 8 * (x % NB));
            }
            __syncwarp();
            return true;
        };
        ok = warp_wait(q_full, 0) && scores(0) && (tiles.count < 2 || scores(1));
        auto products = [&](auto two_parts) {
            for (int x = 0; x < tiles.count && ok; ++x) {
                const int s = x % S::stages;
                ok = warp_wait(p_full + 8 * (x % NB), (x / NB) & 1) && warp_wait(v_full + 8 * s, (x / S::stages) & 1);
                if (!ok) break;
                tc_after();
                const uint64_t dvs = moved(dv, s * S::kv_bytes);
                if (leader) {
#pragma unroll
                    for (int kk = 0; kk < kKeys / 16; ++kk)
                        mma_ts(tm + S::o_col, tm + (x % NB) * kKeys + kk * 8, moved(dvs, kk * 2048), kind_o, x > 0 || kk > 0);
                    if (two_parts.value) {
#pragma unroll
                        for (int kk = 0; kk < kKeys / 16; ++kk)
                            mma_ts(tm + S::o_col, tm + (x % NB) * kKeys + kKeys / 2 + kk * 8, moved(dvs, kk * 2048), kind_o, true);
                    }
                    mma_commit(v_free + 8 * s);
                    mma_commit(o_done);
                }
                __syncwarp();
                if (x + NB < tiles.count) ok = scores(x + NB);
            }
        };
        if (fine) products(std::true_type());
        else products(std::false_type());
        if (leader) {
            mma_commit(o_last);
            if (!ok) report(a.error);
        }
    } else {  // one row each
        const int i = i0 + tid;
        const uint32_t mine = tm + ((uint32_t)(warp * 32) << 16);
        float m = -INFINITY, l = 0.f;  // m: the maximum in use, in scores
        auto softmax = [&](auto two_parts) {
            for (int x = 0; x < tiles.count; ++x) {
                const int j0 = tiles.at(x) * kKeys;
                ok = mbar_wait(s_full + 8 * (x % NB), (x / NB) & 1);
                if (!__all_sync(0xffffffffu, ok)) break;
                tc_after();
                const uint32_t at = mine + (x % NB) * kKeys;
                // every row of the tile sees every key, unless the tile crosses the diagonal or the window's edge
                const bool whole = j0 + kKeys - 1 <= i0 && (i0 + kRows - 1 - j0 < a.window || j0 + kKeys <= a.sinks);
                uint32_t on[2] = {0xffffffffu, 0xffffffffu};
                if (!whole) on[0] = keys_of_row(i, j0, a.window, a.sinks), on[1] = keys_of_row(i, j0 + 32, a.window, a.sinks);
                auto mask = [&](uint32_t *u, int half) {
                    if (whole) return;
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (!(on[half] & (1u << c))) u[c] = 0xff800000u;  // minus infinity
                };
                uint32_t u[2][32];
                float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                auto highest = [&](const uint32_t *v) {
#pragma unroll
                    for (int c = 0; c < 32; ++c) tops[c % 4] = fmaxf(tops[c % 4], __uint_as_float(v[c]));
                };
                tc_ld32(at, u[0]);
                tc_ld32(at + 32, u[1]);
                tc_wait_ld(u[0]);
                tc_touch(u[1]);
#pragma unroll
                for (int half = 0; half < 2; ++half) mask(u[half], half), highest(u[half]);
                const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                float turn = 1.f;
                if (m == -INFINITY) {
                    m = top;  // nothing of this row is in O yet
                } else if ((top - m) * a.scale_log2 > 8.f) {
                    turn = exp2_fast((m - top) * a.scale_log2);
                    l *= turn;
                    m = top;
                }
                if (__any_sync(0xffffffffu, turn != 1.f)) {
                    // until the previous product is in O (these scores were queued behind the one before it)
                    ok = mbar_wait(o_done, (x - 1) & 1);
                    if (!__all_sync(0xffffffffu, ok)) break;
                    tc_after();
#pragma unroll
                    for (int c = 0; c < DP; c += 32) {
                        uint32_t w[32];
                        tc_ld32(mine + S::o_col + c, w);
                        tc_wait_ld(w);
#pragma unroll
                        for (int e = 0; e < 32; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) * turn);
                        tc_st32(mine + S::o_col + c, w);
                    }
                }
                const float off = m == -INFINITY ? 0.f : m * a.scale_log2;
                const uint64_t scale2 = two(a.scale_log2, a.scale_log2), off2 = two(-off, -off);
                uint64_t sum[4] = {};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t *v = u[half];
                    uint32_t p[16];
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        float p0, p1;
                        apart(fma_two(two(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), scale2, off2), p0, p1);
                        p0 = exp2_fast(p0), p1 = exp2_fast(p1);
                        sum[(c / 2) % 4] = add_two(sum[(c / 2) % 4], two(p0, p1));
                        p[c / 2] = pack2(p0, p1, T());
                        if (two_parts.value) v[c] = __float_as_uint(p0), v[c + 1] = __float_as_uint(p1);
                    }
                    tc_st16(at + half * 16, p);  // over scores that have been read
                    if (two_parts.value) {
#pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            float h0, h1;
                            unpack2(p[c / 2], h0, h1, T());
                            p[c / 2] = pack2(__uint_as_float(v[c]) - h0, __uint_as_float(v[c + 1]) - h1, T());
                        }
                        tc_st16(at + kKeys / 2 + half * 16, p);
                    }
                }
                float s0, s1;
                apart(add_two(add_two(sum[0], sum[1]), add_two(sum[2], sum[3])), s0, s1);
                l += s0 + s1;
                // keys behind the sequence meet p = 0, but what they hold may be infinite: their values are zeroed
                if (n < a.T && j0 + kKeys > n) {
                    const int s = x % S::stages;
                    ok = mbar_wait(v_full + 8 * s, (x / S::stages) & 1);
                    if (!__all_sync(0xffffffffu, ok)) break;
                    constexpr int C = DP / 8;
                    const int first = n - j0;
                    for (int e = tid; e < (kKeys - first) * C; e += kRows) {
                        const int r = first + e / C, c = e % C;
                        const uint32_t dst = sv + s * S::kv_bytes + (c / 8) * kKeys * 128 + r * 128 + (c % 8) * 16;
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(0) : "memory");
                    }
                    fence_async();
                    __syncwarp();
                }
                tc_wait_st();
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 8 * (x % NB));
            }
        };
        if (fine) softmax(std::true_type());
        else softmax(std::false_type());
        if (ok) ok = mbar_wait(o_last, 0);
        if (__all_sync(0xffffffffu, ok)) {
            tc_after();
            const bool live = i < n;
            const float inv = l > 0.f ? 1.f / l : 0.f;
            // rows go through shared memory (the queries' place, and the keys' for what rounding takes) so that stores are
            // whole rows
            const uint32_t row = sq + tid * 128, rest = sk + tid * 128;
            static_assert(S::stages * S::kv_bytes >= S::q_bytes);
#pragma unroll
            for (int c = 0; c < DP; c += 32) {
                uint32_t w[32];
                tc_ld32(mine + S::o_col + c, w);
                tc_wait_ld(w);
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    float f[8];
                    uint32_t y[4];
#pragma unroll
                    for (int k = 0; k < 8; ++k) f[k] = live && l != 0.f ? __uint_as_float(w[e + k]) * inv : 0.f;
#pragma unroll
                    for (int k = 0; k < 4; ++k) y[k] = pack2(f[2 * k], f[2 * k + 1], T());
                    const uint32_t to = (c / 64) * kRows * 128 + ((((c % 64 + e) / 8) ^ (tid & 7)) * 16);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + to), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]) : "memory");
                    if (i0 < a.rest_rows) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) y[k] = pack2(rest_of<T>(f[2 * k]), rest_of<T>(f[2 * k + 1]), T());
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(rest + to), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]) : "memory");
                    }
                }
            }
            __syncwarp();
            constexpr int C = DP / 8;
            for (int e = lane; e < 32 * C; e += 32) {
                const int r = warp * 32 + e / C, c = e % C;
                const uint32_t from = (c / 8) * kRows * 128 + r * 128 + (((c % 8) ^ (r & 7)) * 16);
                if (i0 + r >= a.T || c * 8 >= a.D) continue;
                auto copy = [&](uint32_t src, char *dst) {
                    uint4 y;
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w) : "r"(src));
                    *reinterpret_cast<uint4 *>(dst + c * 16) = y;
                };
                copy(sq + from, a.o + b * a.ob + (int64_t)(i0 + r) * a.ot + h * a.oh);
                if (i0 + r < a.rest_rows) copy(sk + from, a.rest + b * a.rb + (int64_t)(i0 + r) * a.rt + h * a.rh);
            }
            if (a.lse && i < a.T) a.lse[((int64_t)b * a.H + h) * a.lse_row + i] = live && l != 0.f ? fmaf(m, a.scale_log2, log2f(l)) : 0.f;  // NaN stays
        } else if (lane == 0) {
            report(a.error);
        }
        tc_before();
    }
    __syncwarp();
    __syncthreads();
    if (warp == 5) tmem_free<S::columns>(tm);
}

template <typename T, int DP> int launch(const cail_ops_attention_args *c, const AttnArgs &a, cudaStream_t st) {
    using S = Shape<DP>;
    Maps maps;
    if (int rc = tensor_map(&maps.q, c->q, c->type, a.B, a.T, a.H, a.D, kRows)) return rc;
    if (int rc = tensor_map(&maps.k, c->k, c->type, a.B, a.T, a.Hkv, a.D, kKeys)) return rc;
    if (int rc = tensor_map(&maps.v, c->v, c->type, a.B, a.T, a.Hkv, a.D, kKeys)) return rc;
    cudaError_t e = cudaFuncSetAttribute(tc_forward_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem);
    if (e != cudaSuccess) return fail(CAIL_OPS_ECUDA, "window attention: %s", cudaGetErrorString(e));
    tc_forward_kernel<T, DP><<<dim3(a.H, a.B, (a.T + kRows - 1) / kRows), kThreads, S::smem, st>>>(a, maps);
    return launched("window attention");
}

}  // namespace

// 16-bit elements in rows that TMA can load (16-byte multiples), a positive
// scale (the row maximum is taken before scaling), no more tiles than a grid
// has; and more than 64 tokens: below, rows have few keys, where rounding ds
// costs most, and the other kernels round neither p nor ds.  That is a choice
// for accuracy and costs time, the more the larger the batch: 8 heads of 64,
// forward and backward, 8 x 32 tokens 25 us (19 here), 64 x 64 114 (37), 4096
// x 64 6660 (1730).  Short windows over more tokens are not left to the other
// kernels: 8 x 1024 tokens, 16 heads of 64, window 8, 117 us here, 1130 there.
bool tc_takes(const cail_ops_attention_args *a) {
    if (a->type == CAIL_OPS_F32 || a->D % 8 || !(a->scale > 0.f) || a->T > kMostTiles * kRows || a->T <= 64) return false;
    if (!tma_takes(a->q, a->B, a->T, a->H) || !tma_takes(a->k, a->B, a->T, a->Hkv) || !tma_takes(a->v, a->B, a->T, a->Hkv)) return false;
    return rows_aligned(a->o, a->B, a->T, a->H, 2, 16) && (!a->o_rest.ptr || rows_aligned(a->o_rest, a->B, a->rest_rows, a->H, 2, 16));
}

int tc_forward(const cail_ops_attention_args *c, cudaStream_t st) {
    AttnArgs a = attn_args(c, false);
    if (int rc = earlier_error("window attention")) return rc;
    a.error = device_error_flag();
    if (!a.error) return fail(CAIL_OPS_ECUDA, "window attention: no error word for this device");
    if (c->type == CAIL_OPS_BF16) return a.D <= 64 ? launch<__nv_bfloat16, 64>(c, a, st) : launch<__nv_bfloat16, 128>(c, a, st);
    return a.D <= 64 ? launch<__half, 64>(c, a, st) : launch<__half, 128>(c, a, st);
}

}  // namespace cailops
