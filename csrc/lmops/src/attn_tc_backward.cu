// attn_tc_backward.cu — gradients of window attention on the tensor cores
// (bf16, fp16).
//
// Two kernels of one shape.  A block keeps 128 rows of X and Y in shared
// memory, streams tiles of 64 rows of U and W past them, and for every tile
//   S = X U^T,  dP = Y W^T          (into tensor memory)
//   p = exp2(S - lse), ds = p (dP - delta)   (256 threads, 32 columns each)
//   acc0 += ds U  [, acc1 += p W]   (p and ds from tensor memory)
// where, with i a query and j a key,
//   dq:     X = Q, Y = dO (rows i), U = K, W = V: acc0 = dq; delta = do.o on the way
//   dk, dv: X = K, Y = V (rows j), U = Q, W = dO over the group's heads: acc0 = dk, acc1 = dv
// Seven products instead of the five of a kernel that adds dq with atomics:
// every output is summed by one block in one order, so results do not change
// from run to run.  The sinks' key tiles are seen by all queries; where that
// would make them the last blocks running, their queries are split and the
// parts joined in order by a third kernel.
//
// p and ds are rounded to the input type for their products, all else is
// 32-bit.  fp16 has no range for small gradients, nor for large ones: ds is
// scaled by a power of two, taken back out of the sums.  It comes from a bound
// of |ds| for each row, 2 sum |do| max |v| over the keys that the row sees
// (|ds| <= |do.v| + |do.o|), brought to [2^14, 2^15): the row's own for dq, the
// largest of the rows that see the key for dk.  So nothing overflows, and no
// row or key loses bits to one that it does not meet.  A small kernel goes over
// v for it first (8 x 1024 tokens, 16 heads of 64, window 256, forward and
// backward: 152 us, and 145 with scales from max |do| alone).
//
// D = 64: two blocks per SM, S of the next tile computed under this one's
// softmax (dq: dP too); 8 x 1024 tokens, 16 heads, window 256 and 4 sinks: dq
// 42 us, dk and dv 59, products a fifth of the tensor pipe, the rest a block's
// prologue and epilogue around five to seven tiles.  D = 128: one block per
// SM, two buffers of S and dP; 8192 tokens, 16 query and 4 key heads, window
// 1024 and 16 sinks: dq 128 us, dk and dv 140, products 80 % of the loop.
#include <algorithm>
#include <type_traits>

#include "attn.cuh"
#include "tc.cuh"

namespace cailops {
namespace {

constexpr int kRows = 128, kStream = 64, kMath = 256, kThreads = kMath + 64;

template <int DP, bool DKV> struct Shape {
    static constexpr int panels = DP / 64;
    static constexpr int stages = 3;
    static constexpr int buffers = DP == 64 ? 1 : 2;  // of S and dP
    static constexpr int per_sm = DP == 64 ? 2 : 1;
    static constexpr int chunk = DKV && DP == 64 ? 16 : 32;  // columns at a time, by the registers that two blocks leave
    static constexpr int x_bytes = kRows * DP * 2, u_bytes = kStream * DP * 2;
    static constexpr int vec_bytes = DKV ? 2 * kStream * 4 : 0;  // lse and delta of a tile's queries
    static constexpr int barriers = 1 + 2 * stages + 2 * buffers + 4;
    static constexpr int o_bytes = DKV ? 0 : x_bytes;  // the output's rows, for delta
    static constexpr int smem = 1024 + 2 * x_bytes + stages * (2 * u_bytes + vec_bytes) + o_bytes;
    static constexpr int acc = buffers * 2 * kStream;  // column of acc0; acc1 follows
    // One buffer: S of the next tile is computed as soon as this one's is read, for p and ds go elsewhere: into dP's
    // columns (dk, dv), or ds into columns of its own, so that the next dP is early too (dq).
    static constexpr bool early = buffers == 1, early_dp = early && !DKV;
    static constexpr int ds = acc + DP;
    static constexpr int columns = DP == 64 ? 256 : 512;
};

struct Maps {
    CUtensorMap x, y, u, w, o, rest;
};

struct Extra {
    // fp16: what ds can reach.  Bits of max |v| of a key, and of the largest |ds| that a row can have, over the group's
    // heads: [B, Hkv, T] each.
    unsigned *v_top, *reach;
    SinkParts parts;
};

// the power of two that brings a value whose largest is `bits` to [2^14, 2^15)
__device__ __forceinline__ float amp_of(unsigned bits) {
    const int e = min(max((int)(bits >> 23) - 127, -100), 100);
    return bits == 0 ? 1.f : __uint_as_float((unsigned)(127 + 14 - e) << 23);
}

// The largest of a value per query row (bits of floats of no sign, a sequence's
// n of them) over the rows that see key r0 + k, k < 128, or (KEYS) of a value
// per key over the keys that row r0 + k sees: for k = tid & 127 of kMath
// threads.  With w the window, the rows that see a key are its own to w - 1
// behind it: 256 values side by side, the tile's own rows and the 128 that
// begin max(w, 128) behind its first, over which a maximum of min(w, 128)
// slides (by doubling), and between the two what all 128 meet.  The keys that
// a row sees are the same in mirror image, and the sinks; a sink is seen by
// every row behind it.
template <bool KEYS>
__device__ __forceinline__ unsigned largest_met(const unsigned *values, int r0, int n, int window, int sinks, unsigned (*buf)[kMath], unsigned *shared) {
    const int tid = threadIdx.x, k = tid & 127, w = min(window, n), width = min(w, 128), far = max(w, 128);
    const int at = r0 + k + (KEYS ? (tid < 128 ? -far : 0) : (tid < 128 ? 0 : far));
    unsigned x = at >= 0 && at < n ? values[at] : 0u, common = 0u, behind = 0u;
    buf[0][tid] = x;
    const int from = KEYS ? max(r0 - w + 128, 0) : r0 + 128, to = KEYS ? r0 : min(r0 + w, n);
    for (int i = from + tid; i < to; i += kMath) common = max(common, values[i]);
    if (KEYS)
        for (int i = tid; i < min(sinks, r0); i += kMath) common = max(common, values[i]);
    if (!KEYS && r0 < sinks)
        for (int i = r0 + 128 + tid; i < n; i += kMath) behind = max(behind, values[i]);
    common = __reduce_max_sync(0xffffffffu, common), behind = __reduce_max_sync(0xffffffffu, behind);
    if ((tid & 31) == 0) shared[tid >> 5] = common, shared[kMath / 32 + (tid >> 5)] = behind;
    auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(kMath) : "memory"); };
    meet();
    int now = 0, wide = 1;
    for (; wide * 2 <= width; wide *= 2) {
        x = max(x, tid + wide < kMath ? buf[now][tid + wide] : 0u);
        now ^= 1;
        buf[now][tid] = x;
        meet();
    }
    const int place = KEYS ? 129 + k - width : k;
    unsigned top = max(buf[now][place], buf[now][place + width - wide]);
    const bool sink = !KEYS && r0 + k < sinks;
    for (int i = 0; i < kMath / 32; ++i) top = max(top, max(shared[i], sink ? shared[kMath / 32 + i] : 0u));
    if (sink)
        for (int i = r0 + k; i < min(r0 + 128, n); ++i) top = max(top, values[i]);
    if (KEYS)
        for (int i = r0; i < min(min(sinks, n), r0 + k + 1); ++i) top = max(top, values[i]);
    return top;
}

// fp16: max |v| of every key (what is not finite aside: the rows that see it are not finite either), and zeros for the rows' reach
template <int DP> __global__ void __launch_bounds__(256) v_top_kernel(const AttnArgs a, const Extra ex) {
    constexpr int LANES = DP / 8, ROWS = 256 / LANES;
    const int hk = blockIdx.y, b = blockIdx.z, r = blockIdx.x * ROWS + threadIdx.x / LANES, c = threadIdx.x % LANES * 8;
    float top = 0.f;
    if (r < length_of(a, b) && c < a.D) {
        const Vec<__half, 8> v = *reinterpret_cast<const Vec<__half, 8> *>(a.v + b * a.vb + (int64_t)r * a.vt + hk * a.vh + c * 2);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float f = fabsf(to_f(v.v[e]));
            if (f < INFINITY) top = fmaxf(top, f);
        }
    }
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (c == 0 && r < a.T) {
        const int64_t at = ((int64_t)b * a.Hkv + hk) * a.T + r;
        ex.v_top[at] = __float_as_uint(top), ex.reach[at] = 0u;
    }
}

template <typename T, int DP, bool DKV>
__global__ void __launch_bounds__(kThreads, Shape<DP, DKV>::per_sm)
    tc_backward_kernel(const AttnArgs a, const Extra ex, const __grid_constant__ Maps maps) {
    using S = Shape<DP, DKV>;
    constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
    constexpr int NB = S::buffers, ST = S::stages;
    extern __shared__ char raw[];
    __shared__ __align__(8) uint64_t bars[S::barriers];
    __shared__ uint32_t tmem_at;
    [[maybe_unused]] __shared__ unsigned met[bf ? 1 : 2][bf ? 1 : kMath], met_all[bf ? 1 : 2 * kMath / 32];
    const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
    const uint32_t sx = base, sy = sx + S::x_bytes, su = sy + S::x_bytes, sw = su + S::u_bytes;  // U and W of a stage side by side
    constexpr uint32_t stage_bytes = 2 * S::u_bytes;
    const uint32_t svec = su + ST * stage_bytes, so = svec;
    const uint32_t srest = su + (ST - 1) * stage_bytes;  // dq: what rounding took from the output, in the last stage until its first tile
    static_assert(DKV || stage_bytes == S::x_bytes);
    const uint32_t bar0 = smem_u32(bars);
    const uint32_t x_full = bar0, full = bar0 + 8, free_ = full + 8 * ST, s_full = free_ + 8 * ST, ds_full = s_full + 8 * NB, last = ds_full + 8 * NB, s_read = last + 8, acc_done = s_read + 8, rest_read = acc_done + 8;

    const int tid = threadIdx.x, warp = warp_number(), lane = tid & 31;
    const int b = blockIdx.y, n = length_of(a, b);
    // rows of this block, and the tiles that pass: x = 0 .. count - 1
    int r0, count, h, hk, split = 0, q_begin = 0, q_tiles = 0, first = 0;
    bool parted = false;
    KeyTiles keys(0, 0, 0, 1, 0, kStream);
    if constexpr (DKV) {
        hk = blockIdx.x, h = hk * a.group;
        int tile = blockIdx.z;
        parted = ex.parts.splits > 1 && tile < ex.parts.tiles * ex.parts.splits;
        if (parted) split = tile % ex.parts.splits, tile /= ex.parts.splits;
        else if (ex.parts.splits > 1) tile -= ex.parts.tiles * (ex.parts.splits - 1);
        r0 = tile * kRows;
        int begin, end;
        query_range(r0, r0 + kRows, n, a.window, a.sinks, begin, end);
        q_begin = begin / kStream;
        q_tiles = end > begin ? (end - 1) / kStream + 1 - q_begin : 0;
        count = a.group * q_tiles;
        if (parted) {  // this part of the tiles
            const int per = (count + ex.parts.splits - 1) / ex.parts.splits;
            first = min(count, split * per);
            count = min(count, first + per) - first;
        }
    } else {
        h = blockIdx.x, hk = h / a.group;
        r0 = (gridDim.z - 1 - blockIdx.z) * kRows;  // the longest rows first
        keys = KeyTiles(r0, r0 + kRows, n, a.window, a.sinks, kStream);
        count = keys.count;
    }
    const bool rested = !DKV && r0 < a.rest_rows;  // what rounding took from these rows' output is there
    // a walk over the tiles: the first row of the tile at hand, and its query head (dk, dv)
    struct Walk {
        int x, row, head;
    };
    auto begin_walk = [&] {
        Walk w = {0, 0, h};
        if constexpr (DKV) {
            w.row = q_begin * kStream;
            if (first > 0) w.row += first % q_tiles * kStream, w.head += first / q_tiles;
        }
        if constexpr (!DKV) w.row = keys.at(0) * kStream;
        return w;
    };
    auto step = [&](Walk &w) {
        ++w.x;
        if constexpr (DKV) {
            w.row += kStream;
            if (w.row == (q_begin + q_tiles) * kStream) w.row = q_begin * kStream, ++w.head;
        } else {
            w.row = keys.at(w.x) * kStream;
        }
    };

    if (count == 0) {  // nothing sees or is seen: zeros
        constexpr int C = DP / 8;
        if (DKV && parted) {
            float4 *p = reinterpret_cast<float4 *>(ex.parts.sums) +
                        ((((int64_t)b * a.Hkv + hk) * ex.parts.tiles + r0 / kRows) * ex.parts.splits + split) * (2 * kRows * DP / 4);
            for (int i = tid; i < 2 * kRows * DP / 4; i += kThreads) p[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            return;
        }
        for (int i = tid; i < kRows * C; i += kThreads) {
            const int r = r0 + i / C, d = (i % C) * 8;
            if (r >= a.T || d >= a.D) continue;
            if (DKV) {
                *reinterpret_cast<uint4 *>(a.dk + b * a.dkb + (int64_t)r * a.dkt + hk * a.dkh + d * 2) = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4 *>(a.dv + b * a.dvb + (int64_t)r * a.dvt + hk * a.dvh + d * 2) = make_uint4(0, 0, 0, 0);
            } else {
                *reinterpret_cast<uint4 *>(a.dq + b * a.dqb + (int64_t)r * a.dqt + h * a.dqh + d * 2) = make_uint4(0, 0, 0, 0);
            }
        }
        return;
    }

    auto load = [&](const Walk &w) {
        const int s = w.x % ST, t0 = w.row, th = DKV ? w.head : hk;
        const uint32_t bar = full + 8 * s;
        mbar_expect(bar, 2 * S::u_bytes + S::vec_bytes);
        for (int p = 0; p < S::panels; ++p) {
            tma_load(su + s * stage_bytes + p * kStream * 128, &maps.u, bar, p * 64, t0, th, b);
            tma_load(sw + s * stage_bytes + p * kStream * 128, &maps.w, bar, p * 64, t0, th, b);
        }
        if constexpr (DKV) {
            // 64 values each, which may reach into the next row or the padding behind the last one: those are masked
            const int64_t at = ((int64_t)b * a.H + th) * a.lse_row + t0;
            bulk_load(svec + s * S::vec_bytes, a.lse + at, kStream * 4, bar);
            bulk_load(svec + s * S::vec_bytes + kStream * 4, a.delta + at, kStream * 4, bar);
        }
    };
    Walk walk = begin_walk();
    if (warp == 8 && lane == 0) {
        mbar_init(x_full, 1);
        for (int s = 0; s < ST; ++s) mbar_init(full + 8 * s, 1), mbar_init(free_ + 8 * s, 1);
        for (int s = 0; s < NB; ++s) mbar_init(s_full + 8 * s, 1), mbar_init(ds_full + 8 * s, kMath / 32);
        mbar_init(last, 1), mbar_init(s_read, kMath / 32), mbar_init(acc_done, 1), mbar_init(rest_read, kMath / 32);
        fence_barrier_init();
        // what needs no free slot is on its way before the block has met
        mbar_expect(x_full, 2 * S::x_bytes + S::o_bytes + (rested ? S::x_bytes : 0));
        for (int p = 0; p < S::panels; ++p) tma_load(sx + p * kRows * 128, &maps.x, x_full, p * 64, r0, DKV ? hk : h, b);
        load(walk);
        for (int p = 0; p < S::panels; ++p) {
            tma_load(sy + p * kRows * 128, &maps.y, x_full, p * 64, r0, DKV ? hk : h, b);
            if (!DKV) tma_load(so + p * kRows * 128, &maps.o, x_full, p * 64, r0, h, b);
            if (rested) tma_load(srest + p * kRows * 128, &maps.rest, x_full, p * 64, r0, h, b);
        }
        for (step(walk); walk.x < (DKV ? ST : ST - 1) && walk.x < count; step(walk)) load(walk);
    }
    if (warp == 9) tmem_alloc<S::columns>(smem_u32(&tmem_at));
    __syncwarp();
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tm = tmem_at;
    bool ok = true;

    if (warp == 8) {
        if (lane == 0) {  // the loads that wait for a slot
            for (; walk.x < count; step(walk)) {
                if (walk.x < ST) ok = mbar_wait(rest_read, 0);  // dq: the last stage's first tile
                else ok = mbar_wait(free_ + 8 * (walk.x % ST), ((walk.x / ST) & 1) ^ 1);
                if (!ok) break;
                load(walk);
            }
            if (!ok) {  // gave up: the copies in flight land before the block ends
                report(a.error);
                mbar_wait(x_full, 0);
                for (int y = max(0, walk.x - ST); y < walk.x; ++y) mbar_wait(full + 8 * (y % ST), (y / ST) & 1);
            }
        }
    } else if (warp == 9) {
        // products: the whole warp runs the loop, one lane issues
        const bool leader = elect_one();
        constexpr uint32_t kind_s = mma_kind<bf, kRows, kStream, false>(), kind_acc = mma_kind<bf, kRows, DP, true>();
        const int steps = (a.D + 15) / 16;
        // U and W as operands along their rows (scores) and down them (sums)
        const uint64_t dx = operand(sx, 0), dy = operand(sy, 0), du = operand(su, 0), dw = operand(sw, 0), dut = operand(su, kStream * 128),
                       dwt = operand(sw, kStream * 128);
        // S and dP of a tile; the second of them announces both
        auto scores = [&](int x, bool first, bool second) {
            const int s = x % ST;
            if (first && !warp_wait(full + 8 * s, (x / ST) & 1)) return false;
            tc_after();
            const uint32_t d = tm + (x % NB) * 2 * kStream;
            const uint64_t dus = moved(du, s * stage_bytes), dws = moved(dw, s * stage_bytes);
            if (leader && first) {
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk)
                    if (kk < steps)
                        mma_ss(d, moved(dx, (kk / 4) * kRows * 128 + (kk % 4) * 32), moved(dus, (kk / 4) * kStream * 128 + (kk % 4) * 32), kind_s,
                               kk > 0);
            }
            if (leader && second) {
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk)
                    if (kk < steps)
                        mma_ss(d + kStream, moved(dy, (kk / 4) * kRows * 128 + (kk % 4) * 32),
                               moved(dws, (kk / 4) * kStream * 128 + (kk % 4) * 32), kind_s, kk > 0);
                mma_commit(s_full + 8 * (x % NB));
            }
            __syncwarp();
            return true;
        };
        ok = warp_wait(x_full, 0);
        for (int x = 0; x < NB && x < count && ok; ++x) ok = scores(x, true, true);
        for (int x = 0; x < count && ok; ++x) {
            const int s = x % ST;
            if (S::early && x + 1 < count) {
                ok = warp_wait(s_read, x & 1) && scores(x + 1, true, S::early_dp);
                if (!ok) break;
            }
            ok = warp_wait(ds_full + 8 * (x % NB), (x / NB) & 1);
            if (!ok) break;
            tc_after();
            const uint32_t d = tm + (x % NB) * 2 * kStream;
            if (leader) {
                // p and ds of 16 rows each, 8 columns; in dP's place they alternate
                if constexpr (DKV) {
#pragma unroll
                    for (int kk = 0; kk < kStream / 16; ++kk)
                        mma_ts(tm + S::acc + DP, d + kStream + kk * 16, moved(dwt, s * stage_bytes + kk * 2048), kind_acc, x > 0 || kk > 0);
                }
#pragma unroll
                for (int kk = 0; kk < kStream / 16; ++kk)
                    mma_ts(tm + S::acc, S::early_dp ? tm + S::ds + kk * 8 : d + kStream + kk * 16 + 8, moved(dut, s * stage_bytes + kk * 2048), kind_acc,
                           x > 0 || kk > 0);
                mma_commit(free_ + 8 * s);
                if (S::early_dp) mma_commit(acc_done);
            }
            __syncwarp();
            if (S::early && !S::early_dp && x + 1 < count) ok = scores(x + 1, false, true);
            if (!S::early && x + NB < count) ok = scores(x + NB, true, true);
        }
        if (leader) {
            mma_commit(last);
            if (!ok) report(a.error);
        }
    } else {  // a row and 32 columns each
        const int half = warp >> 2, row = tid & 127, r = r0 + row;
        const uint32_t mine = tm + ((uint32_t)((warp & 3) * 32) << 16);
        float lse = 0.f, delta = 0.f, amp = 1.f;
        if constexpr (!DKV) {
            const int64_t at = ((int64_t)b * a.H + h) * a.lse_row + r;
            if (r < n) lse = a.lse[at];  // on its way while do and o arrive
            [[maybe_unused]] float v_met = 0.f;
            if constexpr (!bf)
                v_met = __uint_as_float(largest_met<true>(ex.v_top + ((int64_t)b * a.Hkv + hk) * a.T, r0, n, a.window, a.sinks, met, met_all));
            ok = warp_wait(x_full, 0);
            if (ok) {
                float size = 0.f;  // sum |do|
                if (r < n) {
#pragma unroll
                    for (int c = 0; c < DP / 8; ++c) {
                        if (c * 8 >= a.D) break;
                        Vec<T, 8> g, o, rest;
                        const uint32_t at = (c / 8) * kRows * 128 + row * 128 + (((c % 8) ^ (row & 7)) * 16);
                        uint4 w;
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(sy + at));
                        *reinterpret_cast<uint4 *>(&g) = w;
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(so + at));
                        *reinterpret_cast<uint4 *>(&o) = w;
                        if (rested)
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(srest + at));
                        else
                            w = make_uint4(0, 0, 0, 0);
                        *reinterpret_cast<uint4 *>(&rest) = w;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float f = to_f(g.v[e]);
                            delta = fmaf(to_f(o.v[e]) + to_f(rest.v[e]), f, delta);
                            if (!bf) size += fabsf(f) < INFINITY ? fabsf(f) : 0.f;  // an infinite gradient scales no other
                        }
                    }
                    if (half == 0) a.delta[at] = delta;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(rest_read);
                if (!bf) {
                    // |do.v| and |do.o| are at most this times |v|, and p at most 1
                    const unsigned most = __float_as_uint(2.f * size * v_met);
                    amp = amp_of(most);
                    if (half == 0 && most) atomicMax(ex.reach + ((int64_t)b * a.Hkv + hk) * a.T + r, most);
                }
            }
        } else if constexpr (!bf) {
            // a scale for every key, from the rows that see it and from no others
            amp = amp_of(largest_met<false>(ex.reach + ((int64_t)b * a.Hkv + hk) * a.T, r0, n, a.window, a.sinks, met, met_all));
        }
        // fp16, dv: p goes into its product 2^15 times as large, as it has no bits left for rows of many keys otherwise
        // (2^-18 is four bits)
        constexpr int lift = DKV && !bf ? 15 : 0;
        const float ds_amp = amp * (1.f / (1 << lift)), delta_amp = delta * ds_amp;
        for (; walk.x < count; step(walk)) {
            const int x = walk.x, t0 = walk.row, s = x % ST;
            if (ok) ok = mbar_wait(s_full + 8 * (x % NB), (x / NB) & 1);
            if (DKV && ok) ok = mbar_wait(full + 8 * s, (x / ST) & 1);  // lse and delta of the tile (done by then)
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_after();
            const uint32_t at = mine + (x % NB) * 2 * kStream + half * 32;
            const int c0 = t0 + half * 32;
            bool whole;
            if (DKV) whole = r0 + kRows - 1 <= t0 && t0 + kStream <= n && (t0 + kStream - 1 - r0 < a.window || r0 + kRows <= a.sinks);
            else whole = t0 + kStream - 1 <= r0 && (r0 + kRows - 1 - t0 < a.window || t0 + kStream <= a.sinks);
            // signs turned where that costs nothing: exp2(-(lse - s)), and -ds = p (delta - dp), put right in the sums' scale
            const uint64_t scale2 = two(-a.scale_log2, -a.scale_log2), minus = two(-ds_amp, -ds_amp);
            constexpr int CH = S::chunk;
            auto math = [&](auto masked) {
                uint32_t on = 0, on_ds = 0;  // which of the 32 are seen; which of them carry ds
                if (masked.value) {
                    on = DKV ? rows_of_key(r, c0, n, a.window, a.sinks) : keys_of_row(r, c0, a.window, a.sinks);
                    on_ds = a.window == 1 && a.sinks == 0 ? 0u : on;
                    if (DKV ? c0 == 0 : r == 0) on_ds &= DKV ? ~1u : 0u;  // row 0 sees one key
                }
                uint32_t us[32];
                tc_ld32(at, us);
#pragma unroll
                for (int c1 = 0; c1 < 32; c1 += CH) {
                    uint32_t ud[CH], pd[CH / 2];
                    [[maybe_unused]] uint32_t pp[CH / 2];
                    tc_ld<CH>(at + kStream + c1, ud);
                    if (c1 == 0) {
                        tc_wait_ld(us);
                        tc_touch_n<CH>(ud);
                        if (S::early) {  // S is read: the next one may come
                            tc_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(s_read);
                        }
                    } else {
                        tc_wait_n<CH>(ud);
                    }
#pragma unroll
                    for (int c = 0; c < CH; c += 4) {
                        uint64_t l2[2] = {two(lse, lse), two(lse, lse)}, d2[2] = {two(delta_amp, delta_amp), two(delta_amp, delta_amp)};
                        if constexpr (DKV) {
                            const uint32_t v = svec + s * S::vec_bytes + (half * 32 + c1 + c) * 4;
                            float l4[4], d4[4];
                            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(l4[0]), "=f"(l4[1]), "=f"(l4[2]), "=f"(l4[3]) : "r"(v));
                            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                         : "=f"(d4[0]), "=f"(d4[1]), "=f"(d4[2]), "=f"(d4[3])
                                         : "r"(v + kStream * 4));
                            l2[0] = two(l4[0], l4[1]), l2[1] = two(l4[2], l4[3]);
                            d2[0] = two(d4[0], d4[1]), d2[1] = two(d4[2], d4[3]);
                            if (!bf) {
                                l2[0] = add_two(l2[0], two(-lift, -lift)), l2[1] = add_two(l2[1], two(-lift, -lift));
                                d2[0] = mul_two(d2[0], two(ds_amp, ds_amp)), d2[1] = mul_two(d2[1], two(ds_amp, ds_amp));
                            }
                        }
                        float p[4], d[4];
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            apart(fma_two(two(__uint_as_float(us[c1 + c + e]), __uint_as_float(us[c1 + c + e + 1])), scale2, l2[e / 2]), p[e], p[e + 1]);
                            p[e] = exp2_fast(-p[e]), p[e + 1] = exp2_fast(-p[e + 1]);
                            const uint64_t t = fma_two(two(__uint_as_float(ud[c + e]), __uint_as_float(ud[c + e + 1])), minus, d2[e / 2]);
                            apart(mul_two(t, two(p[e], p[e + 1])), d[e], d[e + 1]);
                        }
                        if (masked.value) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if (!(on & (1u << (c1 + c + e)))) p[e] = 0.f;
                                if (!(on_ds & (1u << (c1 + c + e)))) d[e] = 0.f;
                            }
                        }
                        if constexpr (DKV) pp[c / 2] = pack2(p[0], p[1], T()), pp[c / 2 + 1] = pack2(p[2], p[3], T());
                        pd[c / 2] = pack2(d[0], d[1], T()), pd[c / 2 + 1] = pack2(d[2], d[3], T());
                    }
                    if (S::early_dp && c1 == 0 && x > 0) {  // ds of the tile before has been used
                        if (ok) ok = mbar_wait(acc_done, (x - 1) & 1);
                        __syncwarp();
                        tc_after();
                    }
                    // over values that are in registers by now
#pragma unroll
                    for (int k = 0; k < CH / 16; ++k) {
                        const uint32_t to = S::early_dp ? mine + S::ds + half * 16 + c1 / 2 + k * 8 : at + kStream + c1 + k * 16 + 8;
                        if constexpr (DKV) tc_st8(at + kStream + c1 + k * 16, pp + k * 8);
                        tc_st8(to, pd + k * 8);
                    }
                }
            };
            if (whole) math(std::false_type());
            else math(std::true_type());
            // rows behind the sequence meet zeros, but what they hold may be infinite: they are zeroed
            if (n < a.T && t0 + kStream > n) {
                constexpr int C = DP / 8;
                const int lo = n - t0;
                for (int e = tid; e < (kStream - lo) * C; e += kMath) {
                    const int rr = lo + e / C, c = e % C;
                    const uint32_t off = s * stage_bytes + (c / 8) * kStream * 128 + rr * 128 + (c % 8) * 16;
                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(su + off), "r"(0) : "memory");
                    if (DKV) asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sw + off), "r"(0) : "memory");
                }
                fence_async();
                __syncwarp();
            }
            tc_wait_st();
            tc_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ds_full + 8 * (x % NB));
        }
        if (ok) ok = mbar_wait(last, 0);
        if (__all_sync(0xffffffffu, ok)) {
            tc_after();
            // dq: each half takes its half of the columns; dk and dv: one each
            const uint32_t stage = DKV && half ? sy : sx;
            const uint32_t from = mine + S::acc + (DKV && half ? DP : 0);
            const int c_lo = DKV ? 0 : half * (DP / 2), c_hi = DKV ? DP : c_lo + DP / 2;
            const float by = DKV && half ? 1.f / (1 << lift) : -a.scale / amp;
            const bool live = r < n;
            float *part = nullptr;
            if (DKV && parted)
                part = ex.parts.sums + (((((int64_t)b * a.Hkv + hk) * ex.parts.tiles + r0 / kRows) * ex.parts.splits + split) * 2 + half) * (kRows * DP) + row * DP;
#pragma unroll 1
            for (int c = c_lo; c < c_hi; c += 32) {
                uint32_t w[32];
                tc_ld32(from + c, w);
                tc_wait_ld(w);
                if (DKV && parted) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<float4 *>(part + c + e) =
                            live ? make_float4(__uint_as_float(w[e]) * by, __uint_as_float(w[e + 1]) * by, __uint_as_float(w[e + 2]) * by,
                                               __uint_as_float(w[e + 3]) * by)
                                 : make_float4(0.f, 0.f, 0.f, 0.f);
                    continue;
                }
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    uint32_t y[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        y[k] = live ? pack2(__uint_as_float(w[e + 2 * k]) * by, __uint_as_float(w[e + 2 * k + 1]) * by, T()) : 0u;
                    const int chunk = (c % 64 + e) / 8;
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + (c / 64) * kRows * 128 + row * 128 + ((chunk ^ (row & 7)) * 16)),
                                 "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3])
                                 : "memory");
                }
            }
            __syncwarp();
            if (!(DKV && parted)) {
                char *out = DKV ? (half ? a.dv + b * a.dvb + hk * a.dvh : a.dk + b * a.dkb + hk * a.dkh) : a.dq + b * a.dqb + h * a.dqh;
                const int64_t step = DKV ? (half ? a.dvt : a.dkt) : a.dqt;
                constexpr int C = DKV ? DP / 8 : DP / 16;
                for (int e = lane; e < 32 * C; e += 32) {
                    const int rr = (warp & 3) * 32 + e / C, c = e % C + c_lo / 8;
                    uint4 y;
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w)
                                 : "r"(stage + (c / 8) * kRows * 128 + rr * 128 + (((c % 8) ^ (rr & 7)) * 16)));
                    if (r0 + rr < a.T && c * 8 < a.D) *reinterpret_cast<uint4 *>(out + (int64_t)(r0 + rr) * step + c * 16) = y;
                }
            }
        } else if (lane == 0) {
            report(a.error);
        }
        tc_before();
    }
    __syncwarp();
    __syncthreads();
    if (warp == 9) tmem_free<S::columns>(tm);
}

struct Layout {
    size_t v_top, reach, sums, total;
    SinkParts parts;
};
Layout layout_of(const cail_ops_attention_args *c) {
    Layout l = {};
    l.parts = sink_parts(c, kRows, kStream, (int64_t)sm_count() * (c->D <= 64 ? 2 : 1));
    const size_t values = c->type == CAIL_OPS_F16 ? ((size_t)c->B * c->Hkv * c->T * 4 + 255) / 256 * 256 : 0;
    l.reach = values, l.sums = 2 * values;
    l.total = l.sums + sink_bytes(c, l.parts, kRows, c->D <= 64 ? 64 : 128);
    return l;
}

template <typename T, int DP> int launch(const cail_ops_attention_args *c, AttnArgs a, cudaStream_t st) {
    const Layout l = layout_of(c);
    if (c->workspace_bytes < l.total || (l.total && (!c->workspace || !aligned(c->workspace, 16))))
        return fail(CAIL_OPS_EINVAL, "window attention backward: a workspace of %zu bytes is needed", l.total);
    Extra ex = {};
    ex.v_top = reinterpret_cast<unsigned *>(static_cast<char *>(c->workspace) + l.v_top);
    ex.reach = reinterpret_cast<unsigned *>(static_cast<char *>(c->workspace) + l.reach);
    ex.parts = l.parts;
    ex.parts.sums = reinterpret_cast<float *>(static_cast<char *>(c->workspace) + l.sums);
    // the same arrays with boxes of 128 and of 64 rows
    Maps q = {}, k = {};
    if (int rc = tensor_map(&q.o, c->o, c->type, a.B, a.T, a.H, a.D, kRows)) return rc;
    if (a.rest_rows)
        if (int rc = tensor_map(&q.rest, c->o_rest, c->type, a.B, a.rest_rows, a.H, a.D, kRows)) return rc;
    if (int rc = tensor_map(&q.x, c->q, c->type, a.B, a.T, a.H, a.D, kRows)) return rc;
    if (int rc = tensor_map(&q.y, c->dout, c->type, a.B, a.T, a.H, a.D, kRows)) return rc;
    if (int rc = tensor_map(&q.u, c->k, c->type, a.B, a.T, a.Hkv, a.D, kStream)) return rc;
    if (int rc = tensor_map(&q.w, c->v, c->type, a.B, a.T, a.Hkv, a.D, kStream)) return rc;
    if (int rc = tensor_map(&k.x, c->k, c->type, a.B, a.T, a.Hkv, a.D, kRows)) return rc;
    if (int rc = tensor_map(&k.y, c->v, c->type, a.B, a.T, a.Hkv, a.D, kRows)) return rc;
    if (int rc = tensor_map(&k.u, c->q, c->type, a.B, a.T, a.H, a.D, kStream)) return rc;
    if (int rc = tensor_map(&k.w, c->dout, c->type, a.B, a.T, a.H, a.D, kStream)) return rc;
    const unsigned tiles = (a.T + kRows - 1) / kRows;
    constexpr int sm_q = Shape<DP, false>::smem, sm_k = Shape<DP, true>::smem;
    cudaError_t e = cudaFuncSetAttribute(tc_backward_kernel<T, DP, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, sm_q);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(tc_backward_kernel<T, DP, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, sm_k);
    if (e != cudaSuccess) return fail(CAIL_OPS_ECUDA, "window attention backward: %s", cudaGetErrorString(e));
    if (c->type == CAIL_OPS_F16) {
        constexpr int rows = 256 / (DP / 8);
        v_top_kernel<DP><<<dim3((a.T + rows - 1) / rows, a.Hkv, a.B), 256, 0, st>>>(a, ex);
        if (int rc = launched("window attention backward")) return rc;
    }
    tc_backward_kernel<T, DP, false><<<dim3(a.H, a.B, tiles), kThreads, sm_q, st>>>(a, ex, q);
    if (int rc = launched("window attention backward")) return rc;
    const unsigned blocks = tiles + ex.parts.tiles * (ex.parts.splits - 1);  // at most kMostTiles: sink_parts()
    tc_backward_kernel<T, DP, true><<<dim3(a.Hkv, a.B, blocks), kThreads, sm_k, st>>>(a, ex, k);
    if (int rc = launched("window attention backward")) return rc;
    if (ex.parts.splits == 1) return CAIL_OPS_OK;
    return join<T, DP, kRows>(a, ex.parts, st);
}

}  // namespace

bool tc_takes_backward(const cail_ops_attention_args *a) {
    return tc_takes(a) && tma_takes(a->dout, a->B, a->T, a->H) && tma_takes(a->o, a->B, a->T, a->H) && (!a->o_rest.ptr || tma_takes(a->o_rest, a->B, a->rest_rows, a->H)) && rows_aligned(a->dq, a->B, a->T, a->H, 2, 16) &&
           rows_aligned(a->dk, a->B, a->T, a->Hkv, 2, 16) && rows_aligned(a->dv, a->B, a->T, a->Hkv, 2, 16) && aligned(a->lse, 16) &&
           aligned(a->delta, 16);
}

size_t tc_workspace(const cail_ops_attention_args *c) { return layout_of(c).total; }

int tc_backward(const cail_ops_attention_args *c, cudaStream_t st) {
    AttnArgs a = attn_args(c, true);
    if (int rc = earlier_error("window attention backward")) return rc;
    a.error = device_error_flag();
    if (!a.error) return fail(CAIL_OPS_ECUDA, "window attention backward: no error word for this device");
    if (c->type == CAIL_OPS_BF16) return a.D <= 64 ? launch<__nv_bfloat16, 64>(c, a, st) : launch<__nv_bfloat16, 128>(c, a, st);
    return a.D <= 64 ? launch<__half, 64>(c, a, st) : launch<__half, 128>(c, a, st);
}

}  // namespace cailops
