// ops_rotary.cu — rotary positions on q and k in one launch.
//
// Pair i of a head turns by the angle pos * f_i: a' = m (a cos - b sin),
// b' = m (b cos + a sin).  The angle is formed in 64 bits as full turns and
// reduced to [-1/2, 1/2]; sine and cosine are taken of its 32-bit rounding and
// turned by what that left, so a position of a few hundred thousand costs no
// accuracy and no table of positions is kept.  Each (token, pair) is evaluated
// once per block into shared memory and used by all heads of q and k.  Bound
// by memory: every element is read
// and written once (32767 tokens of 40 heads of 128, float32, interleaved:
// 1.34 GB in 207 us, 6.5 TB/s; 8 x 1024 tokens of 32 heads of 64, bf16: 67 MB
// in 13.6 us).
#include <algorithm>

#include "ops_common.cuh"

namespace cailops {
namespace {

struct Side {
    const char *in;
    char *out;
    int64_t isb, ist, ish, osb, ost, osh;  // bytes
    int heads;
};

struct RotaryArgs {
    Side s[2];
    const void *pos;
    int64_t pos_sb, pos_st;
    const double *turns;
    int64_t tokens;
    int T, D, part, per_block;
    int units, abreast, lanes, head_lanes;  // units of a head, how many of them side by side, times how many (token, head) pairs, of how many heads
    float amplitude;
    int inverse;
};

constexpr int kThreads = 256;
constexpr double kPi = 3.14159265358979323846;

// POS: 0 none (0..T-1), 1 int32, 2 int64.  VB: bytes of a vector.
template <typename T, int VB, bool INTER, int POS>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryArgs a) {
    constexpr int N = VB / (int)sizeof(T);
    using V = Vec<T, N>;
    extern __shared__ float2 cs[];  // [per_block][part / 2]
    const int half = a.part / 2;
    const int64_t first = (int64_t)blockIdx.x * a.per_block;
    const int here = (int)min((int64_t)a.per_block, a.tokens - first);

    for (int i = threadIdx.x; i < here * half; i += kThreads) {
        const int tok = i / half, p = i - tok * half;
        const int64_t g = first + tok, b = g / a.T, t = g - b * a.T;
        int64_t at = t;
        if (POS == 1) at = static_cast<const int32_t *>(a.pos)[b * a.pos_sb + t * a.pos_st];
        if (POS == 2) at = static_cast<const int64_t *>(a.pos)[b * a.pos_sb + t * a.pos_st];
        double turn = (double)at * a.turns[p];
        turn -= rint(turn);
        const float half_turns = (float)(2.0 * turn), left = (float)((2.0 * turn - (double)half_turns) * kPi);
        float s, c;
        sincospif(half_turns, &s, &c);
        const float sine = fmaf(left, c, s), cosine = fmaf(-left, s, c);  // at the angle that was rounded away
        cs[i] = make_float2(cosine * a.amplitude, (a.inverse ? -sine : sine) * a.amplitude);
    }
    __syncthreads();

    // A unit of a head is N pairs of the half layout (two vectors), one vector
    // of the interleaved one (one pair where vectors are single elements), or
    // one vector of the part that passes.
    const int l = threadIdx.x / a.abreast;
    if (l >= a.lanes) return;
    const int heads = a.s[0].heads + a.s[1].heads;
    const int rotated = INTER ? (N > 1 ? a.part / N : half) : half / N;
    if constexpr (INTER && N > 1) {
        // thread = (unit, token, head lane): it keeps its unit's angles of a
        // token and goes over the heads, four on their way at a time (32767
        // tokens of 40 heads of 128, float32: 314 us one at a time, 207 so)
        constexpr int ANGLES = N / 2, U = 4;
        for (int u = threadIdx.x % a.abreast; u < a.units; u += a.abreast) {
            const bool pass = u >= rotated;
            const int at = pass ? a.part + (u - rotated) * N : u * N;
            for (int tok = l / a.head_lanes; tok < here; tok += a.lanes / a.head_lanes) {
                const int64_t g = first + tok, b = g / a.T, t = g - b * a.T;
                float2 w[ANGLES];
                if (!pass)
#pragma unroll
                    for (int i = 0; i < ANGLES; ++i) w[i] = cs[tok * half + u * ANGLES + i];
                const char *in[2] = {a.s[0].in + b * a.s[0].isb + t * a.s[0].ist, a.s[1].in + b * a.s[1].isb + t * a.s[1].ist};
                char *out[2] = {a.s[0].out + b * a.s[0].osb + t * a.s[0].ost, a.s[1].out + b * a.s[1].osb + t * a.s[1].ost};
                for (int h0 = l % a.head_lanes; h0 < heads; h0 += U * a.head_lanes) {
                    V x[U];
#pragma unroll
                    for (int i = 0; i < U; ++i) {
                        const int h = h0 + i * a.head_lanes;
                        if (h < heads) {
                            const T *p = reinterpret_cast<const T *>(h < a.s[0].heads ? in[0] + h * a.s[0].ish : in[1] + (h - a.s[0].heads) * a.s[1].ish);
                            x[i] = *reinterpret_cast<const V *>(p + at);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < U; ++i) {
                        const int h = h0 + i * a.head_lanes;
                        if (h >= heads) break;
                        T *p = reinterpret_cast<T *>(h < a.s[0].heads ? out[0] + h * a.s[0].osh : out[1] + (h - a.s[0].heads) * a.s[1].osh);
                        if (!pass) {
#pragma unroll
                            for (int k = 0; k < ANGLES; ++k) {
                                const float f0 = to_f(x[i].v[2 * k]), f1 = to_f(x[i].v[2 * k + 1]);
                                x[i].v[2 * k] = from_f<T>(f0 * w[k].x - f1 * w[k].y);
                                x[i].v[2 * k + 1] = from_f<T>(f1 * w[k].x + f0 * w[k].y);
                            }
                        }
                        *reinterpret_cast<V *>(p + at) = x[i];
                    }
                }
            }
        }
    } else {
        // thread = (unit, lane over (token, head)); two vectors on their way
        // are enough here, and more cost the occupancy that feeds the memory
        // (the same in bf16, all 128 rotated: 115 us, 148 or more with two units)
        int tok = l / heads, h = l - tok * heads;
        const int dt = a.lanes / heads, dh = a.lanes - dt * heads;
        int64_t b = (first + tok) / a.T;
        int t = (int)(first + tok - b * a.T);
        while (tok < here) {
            const Side &s = a.s[h >= a.s[0].heads];
            const int hh = h >= a.s[0].heads ? h - a.s[0].heads : h;
            const T *in = reinterpret_cast<const T *>(s.in + b * s.isb + t * s.ist + hh * s.ish);
            T *out = reinterpret_cast<T *>(s.out + b * s.osb + t * s.ost + hh * s.osh);
            const float2 *w = cs + tok * half;
            for (int u = threadIdx.x % a.abreast; u < a.units; u += a.abreast) {
                if (u >= rotated) {
                    const int at = a.part + (u - rotated) * N;
                    *reinterpret_cast<V *>(out + at) = *reinterpret_cast<const V *>(in + at);
                } else {
                    const int xo = INTER ? 2 * u : u * N, yo = INTER ? 2 * u + 1 : half + u * N;
                    V x = *reinterpret_cast<const V *>(in + xo);
                    V y = *reinterpret_cast<const V *>(in + yo);
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const float2 c = w[u * N + i];
                        const float p = to_f(x.v[i]), q = to_f(y.v[i]);
                        x.v[i] = from_f<T>(p * c.x - q * c.y);
                        y.v[i] = from_f<T>(q * c.x + p * c.y);
                    }
                    *reinterpret_cast<V *>(out + xo) = x;
                    *reinterpret_cast<V *>(out + yo) = y;
                }
            }
            tok += dt, t += dt, h += dh;
            if (h >= heads) h -= heads, ++tok, ++t;
            if (t >= a.T) b += t / a.T, t %= a.T;
        }
    }
}

template <typename T, int VB, bool INTER>
void launch(const RotaryArgs &a, int pos, unsigned grid, size_t smem, cudaStream_t st) {
    if (pos == 0) rotary_kernel<T, VB, INTER, 0><<<grid, kThreads, smem, st>>>(a);
    if (pos == 1) rotary_kernel<T, VB, INTER, 1><<<grid, kThreads, smem, st>>>(a);
    if (pos == 2) rotary_kernel<T, VB, INTER, 2><<<grid, kThreads, smem, st>>>(a);
}

template <typename T, int VB>
void launch(const RotaryArgs &a, bool inter, int pos, unsigned grid, size_t smem, cudaStream_t st) {
    if (inter) launch<T, VB, true>(a, pos, grid, smem, st);
    else launch<T, VB, false>(a, pos, grid, smem, st);
}

}  // namespace
}  // namespace cailops

extern "C" int cail_ops_rotary(const cail_ops_rotary_args *r, cail_ops_stream stream) {
    using namespace cailops;
    const size_t size = type_size(r->type);
    const int Hk = r->k.ptr ? r->Hk : 0;
    if (r->type < CAIL_OPS_F32 || r->type > CAIL_OPS_F16) return fail(CAIL_OPS_EINVAL, "rotary: unknown element type %d", r->type);
    if (r->B < 0 || r->T < 0 || r->H < 0 || Hk < 0 || r->D < 2 || r->D > 1024 || r->part < 2 || r->part > r->D || r->part % 2)
        return fail(CAIL_OPS_EINVAL, "rotary: bad sizes (B %d T %d H %d Hk %d D %d part %d)", r->B, r->T, r->H, Hk, r->D, r->part);
    const int64_t tokens = (int64_t)r->B * r->T;
    if (tokens == 0 || r->H + Hk == 0) return CAIL_OPS_OK;
    const bool in_place = r->q_out.ptr == r->q.ptr && (!Hk || r->k_out.ptr == r->k.ptr);

    // the widest vector that every row allows
    size_t vb = 16;
    auto fits = [&](size_t v) {
        const int n = (int)(v / size);
        const bool sizes = r->interleaved ? r->part % n == 0 : (r->part / 2) % n == 0;
        return sizes && (in_place || (r->D - r->part) % n == 0) &&
               rows_aligned(r->q, r->B, r->T, r->H, size, v) && rows_aligned(r->q_out, r->B, r->T, r->H, size, v) &&
               (!Hk || (rows_aligned(r->k, r->B, r->T, Hk, size, v) && rows_aligned(r->k_out, r->B, r->T, Hk, size, v)));
    };
    while (vb > size && !fits(vb)) vb /= 2;

    RotaryArgs a = {};
    auto side = [&](Side &s, const cail_ops_bthd &in, const cail_ops_bthd &out, int heads) {
        s.in = static_cast<const char *>(in.ptr);
        s.out = static_cast<char *>(out.ptr);
        s.isb = in.sb * (int64_t)size, s.ist = in.st * (int64_t)size, s.ish = in.sh * (int64_t)size;
        s.osb = out.sb * (int64_t)size, s.ost = out.st * (int64_t)size, s.osh = out.sh * (int64_t)size;
        s.heads = heads;
    };
    side(a.s[0], r->q, r->q_out, r->H);
    if (Hk) side(a.s[1], r->k, r->k_out, Hk);
    a.pos = r->positions;
    a.pos_sb = r->pos_sb;
    a.pos_st = r->pos_st;
    a.turns = r->turns;
    a.tokens = tokens;
    a.T = r->T, a.D = r->D, a.part = r->part;
    a.amplitude = r->amplitude;
    a.inverse = r->inverse;
    const int n = (int)(vb / size);
    a.units = (r->interleaved && n > 1 ? r->part / n : r->part / 2 / n) + (in_place ? 0 : (r->D - r->part) / n);
    a.abreast = a.units < kThreads ? a.units : kThreads;
    a.lanes = kThreads / a.abreast;
    // Tokens per block: four rounds of its threads (eight of the interleaved layout's), and an angle for every
    // thread (one token of 40 heads of 128 a block left most threads waiting
    // for the others' sines: 32767 such tokens 350 us); at most 16 KB of
    // angles, fewer tokens when that leaves SMs without a block.
    const int64_t heads = r->H + Hk, half = r->part / 2, sms = sm_count();
    const int64_t per_round = (int64_t)a.units * heads;
    int64_t per = std::max(((r->interleaved ? 8 : 4) * kThreads + per_round - 1) / per_round, (kThreads + half - 1) / half);
    per = std::min(per, std::max<int64_t>(1, 2048 / half));
    const int64_t spread = (tokens + 2 * sms - 1) / (2 * sms + 1);
    per = std::min(per, std::max<int64_t>(1, spread));
    a.per_block = (int)per;
    // interleaved vectors: as many lanes to a token as its block's tokens leave,
    // and whole tokens only (a head that two lanes took would turn twice in place)
    a.head_lanes = (int)std::min<int64_t>(std::min<int64_t>(a.lanes, heads), std::max<int64_t>(1, a.lanes / per));
    if (r->interleaved && n > 1) a.lanes = a.lanes / a.head_lanes * a.head_lanes;
    const int64_t grid = (tokens + per - 1) / per;
    if (grid > 0x7fffffff) return fail(CAIL_OPS_EINVAL, "rotary: too many tokens");
    const size_t smem = (size_t)per * (r->part / 2) * sizeof(float2);
    const int pos = !r->positions ? 0 : r->positions64 ? 2 : 1;
    auto st = static_cast<cudaStream_t>(stream);
    const bool it = r->interleaved != 0;
    const unsigned gr = (unsigned)grid;
    if (r->type == CAIL_OPS_F32) {
        if (vb == 16) launch<float, 16>(a, it, pos, gr, smem, st);
        else if (vb == 8) launch<float, 8>(a, it, pos, gr, smem, st);
        else launch<float, 4>(a, it, pos, gr, smem, st);
    } else if (r->type == CAIL_OPS_BF16) {
        if (vb == 16) launch<__nv_bfloat16, 16>(a, it, pos, gr, smem, st);
        else if (vb == 8) launch<__nv_bfloat16, 8>(a, it, pos, gr, smem, st);
        else if (vb == 4) launch<__nv_bfloat16, 4>(a, it, pos, gr, smem, st);
        else launch<__nv_bfloat16, 2>(a, it, pos, gr, smem, st);
    } else {
        if (vb == 16) launch<__half, 16>(a, it, pos, gr, smem, st);
        else if (vb == 8) launch<__half, 8>(a, it, pos, gr, smem, st);
        else if (vb == 4) launch<__half, 4>(a, it, pos, gr, smem, st);
        else launch<__half, 2>(a, it, pos, gr, smem, st);
    }
    return launched("rotary");
}
