// cail_ops_torch — PyTorch binding of the language-model operators.
//
// Python hands over the path of libcail_ops.so (load()); the kernels are
// reached through its C interface (cail_ops.h).  This file checks arguments,
// allocates outputs through torch's allocator, takes the current stream of
// the tensors' device and provides the backward passes.  Argument errors are
// ValueError or TypeError and come before anything touches a device.
#include <ATen/MemoryOverlap.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <optional>
#include <string>
#include <vector>

#include "../lmops/include/cail_ops.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// Messages are put together without iostreams: this file and torch may be
// built against different C++ runtimes, whose streams do not mix.
void put(std::string &s, const char *x) { s += x; }
void put(std::string &s, const std::string &x) { s += x; }
void put(std::string &s, int64_t x) { s += std::to_string(x); }
void put(std::string &s, int x) { s += std::to_string(x); }
void put(std::string &s, double x) { s += std::to_string(x); }
void put(std::string &s, at::ScalarType x) { s += at::toString(x); }
void put(std::string &s, const at::Device &x) { s += x.str(); }
void put(std::string &s, at::IntArrayRef x) {
    s += '[';
    for (size_t i = 0; i < x.size(); ++i) s += (i ? ", " : "") + std::to_string(x[i]);
    s += ']';
}
template <typename... A> std::string cat(const A &...a) {
    std::string s;
    (put(s, a), ...);
    return s;
}
#define VALUE_CHECK(cond, ...) TORCH_CHECK_VALUE(cond, cat(__VA_ARGS__))
#define TYPE_CHECK(cond, ...) TORCH_CHECK_TYPE(cond, cat(__VA_ARGS__))

struct Lib {
    decltype(&cail_ops_rotary) rotary = nullptr;
    decltype(&cail_ops_window_attention) attention = nullptr;
    decltype(&cail_ops_window_attention_workspace) workspace = nullptr;
    decltype(&cail_ops_window_attention_backward) attention_backward = nullptr;
    decltype(&cail_ops_window_attention_decode) decode = nullptr;
    decltype(&cail_ops_distill) distill = nullptr;
    decltype(&cail_ops_distill_backward) distill_backward = nullptr;
    decltype(&cail_ops_last_error) last_error = nullptr;
    decltype(&cail_ops_launches) launches = nullptr;
} L;

void load(const std::string &path) {
    void *h = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
    TORCH_CHECK(h, cat("cail_ops_torch: ", dlerror()));
    auto get = [&](auto &f, const char *name) {
        f = reinterpret_cast<std::decay_t<decltype(f)>>(dlsym(h, name));
        TORCH_CHECK(f, cat("cail_ops_torch: ", path, " has no ", name));
    };
    get(L.rotary, "cail_ops_rotary");
    get(L.attention, "cail_ops_window_attention");
    get(L.workspace, "cail_ops_window_attention_workspace");
    get(L.attention_backward, "cail_ops_window_attention_backward");
    get(L.decode, "cail_ops_window_attention_decode");
    get(L.distill, "cail_ops_distill");
    get(L.distill_backward, "cail_ops_distill_backward");
    get(L.last_error, "cail_ops_last_error");
    get(L.launches, "cail_ops_launches");
}

constexpr int64_t kIntMax = std::numeric_limits<int>::max();

void done(int rc) {
    if (rc == CAIL_OPS_OK) return;
    VALUE_CHECK(rc != CAIL_OPS_EINVAL, L.last_error());
    TORCH_CHECK(false, L.last_error());
}

int type_of(const Tensor &t, const char *who, const char *what) {
    switch (t.scalar_type()) {
        case at::kFloat: return CAIL_OPS_F32;
        case at::kBFloat16: return CAIL_OPS_BF16;
        case at::kHalf: return CAIL_OPS_F16;
        default: TYPE_CHECK(false, who, ": ", what, " must be float32, bfloat16 or float16, not ", t.scalar_type());
    }
}

// after all other checks: the tensors' device is a CUDA device, the same for all
void same_device(const char *who, const Tensor &first, std::initializer_list<const Tensor *> others) {
    VALUE_CHECK(first.is_cuda(), who, ": needs CUDA tensors, not ", first.device());
    for (const Tensor *t : others)
        VALUE_CHECK(!t->defined() || t->device() == first.device(), who, ": tensors on ", first.device(), " and ", t->device());
}

// what a kernel that is handed a pointer would get wrong without a word: a
// layout without strides, a negation still to be done, a forward-mode tangent
void plain(const char *who, std::initializer_list<const Tensor *> ts) {
    for (const Tensor *t : ts) {
        if (!t->defined()) continue;
        VALUE_CHECK(t->layout() == at::kStrided, who, ": needs strided tensors");
        VALUE_CHECK(!t->is_neg(), who, ": a tensor whose negation is still to be done; call resolve_neg()");
        TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), cat(who, ": has no forward-mode derivative"));
    }
}

cail_ops_stream stream_of(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// rows whose elements lie side by side; a copy where they do not
Tensor rows(const Tensor &t) { return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

// 16-bit rows that the tensor-core kernels' tile loads take: 16-byte
// boundaries, no repeated rows
bool tiled(const Tensor &t) {
    auto ok = [&](int64_t i) { return t.size(i) == 1 || (t.stride(i) > 0 && t.stride(i) % 8 == 0); };
    return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && (t.size(3) == 1 || t.stride(3) == 1) && ok(0) && ok(1) && ok(2);
}
// The same values in rows that they take, where that pays: a copy costs one
// pass over the tensor, the other kernels many times the products' time.  The
// same bound holds for heads that are padded to a multiple of 8.  Copies
// against the other kernels, causal, bf16, forward and backward, GPU time: rows
// off 16 bytes, heads of 64: 129 tokens of one head 29 and 72 us, 1000 tokens
// 62 and 387, 8 x 129 tokens of 16 heads 37 and 173; heads of 33: 45 and 74,
// 80 and 397, 58 and 172.
constexpr int64_t kCopyFrom = 128;  // tokens
Tensor for_tiles(const Tensor &t) {
    if (t.scalar_type() == at::kFloat || t.size(3) % 8 || t.size(1) <= kCopyFrom || t.numel() == 0 || tiled(t)) return t;
    return t.clone(at::MemoryFormat::Contiguous);
}

cail_ops_bthd view(const Tensor &t) {
    if (t.dim() == 3) return {t.data_ptr(), t.stride(0), 0, t.stride(1)};
    return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}

bool wants_grad(std::initializer_list<const Tensor *> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// autograd takes a missing tensor as an empty optional, the code below as an undefined tensor
Tensor or_none(const std::optional<Tensor> &t) { return t.has_value() ? *t : Tensor(); }
std::optional<Tensor> maybe(const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// ------------------------------------------------------------------ rotary

struct RotaryHow {
    Tensor turns, positions;
    int64_t part;
    bool interleaved, inverse;
    double amplitude;
};

void rotary_check(const char *who, const Tensor &q, const Tensor &k, const RotaryHow &w) {
    plain(who, {&q, &k, &w.positions});
    VALUE_CHECK(q.dim() == 4, who, ": q must be [B, T, H, D], got ", q.sizes());
    for (int64_t i = 0; i < 3; ++i)
        VALUE_CHECK(q.size(i) <= kIntMax && (!k.defined() || k.dim() != 4 || k.size(i) <= kIntMax), who, ": at most 2^31 - 1 sequences, tokens and heads");
    type_of(q, who, "q");
    VALUE_CHECK(w.part <= q.size(3), who, ": the plan rotates ", w.part, " elements of heads of ", q.size(3));
    VALUE_CHECK(q.size(3) <= 1024, who, ": heads of at most 1024 elements");
    if (k.defined()) {
        VALUE_CHECK(k.dim() == 4 && k.size(0) == q.size(0) && k.size(1) == q.size(1) && k.size(3) == q.size(3), who,
                          ": k must be [B, T, Hk, D] with q's B, T and D, got ", k.sizes(), " for q ", q.sizes());
        TYPE_CHECK(k.scalar_type() == q.scalar_type(), who, ": q and k differ in type");
    }
    if (w.positions.defined()) {
        const Tensor &p = w.positions;
        TYPE_CHECK(p.scalar_type() == at::kLong || p.scalar_type() == at::kInt, who, ": positions must be int32 or int64");
        VALUE_CHECK((p.dim() == 1 && p.size(0) == q.size(1)) || (p.dim() == 2 && p.size(0) == q.size(0) && p.size(1) == q.size(1)), who,
                          ": positions must be [T] or [B, T], got ", p.sizes(), " for q ", q.sizes());
    }
    same_device(who, q, {&k, &w.turns, &w.positions});
}

void rotary_launch(const Tensor &q, const Tensor &k, const Tensor &qo, const Tensor &ko, const RotaryHow &w) {
    c10::cuda::CUDAGuard guard(q.device());
    cail_ops_rotary_args a = {};
    a.type = type_of(q, "rotary", "q");
    a.B = (int)q.size(0), a.T = (int)q.size(1), a.H = (int)q.size(2), a.D = (int)q.size(3);
    a.part = (int)w.part;
    a.interleaved = w.interleaved, a.inverse = w.inverse;
    a.q = view(q), a.q_out = view(qo);
    if (k.defined()) a.Hk = (int)k.size(2), a.k = view(k), a.k_out = view(ko);
    if (w.positions.defined()) {
        const Tensor &p = w.positions;
        a.positions = p.data_ptr();
        a.positions64 = p.scalar_type() == at::kLong;
        a.pos_sb = p.dim() == 2 ? p.stride(0) : 0;
        a.pos_st = p.stride(p.dim() - 1);
    }
    a.turns = w.turns.data_ptr<double>();
    a.amplitude = (float)w.amplitude;
    done(L.rotary(&a, stream_of(q)));
}

variable_list rotary_out(const Tensor &q, const Tensor &k, const RotaryHow &w) {
    const Tensor qr = rows(q), kr = k.defined() ? rows(k) : k;
    Tensor qo = at::empty(q.sizes(), q.options()), ko = k.defined() ? at::empty(k.sizes(), k.options()) : Tensor();
    if (q.numel() || (k.defined() && k.numel())) rotary_launch(qr, kr, qo, ko, w);
    return k.defined() ? variable_list{qo, ko} : variable_list{qo};
}

struct RotaryFn : torch::autograd::Function<RotaryFn> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const std::optional<Tensor> &k, const Tensor &turns,
                                 const std::optional<Tensor> &positions_, int64_t part, bool interleaved, bool inverse, double amplitude) {
        const Tensor positions = or_none(positions_);
        ctx->save_for_backward({turns, positions});
        ctx->saved_data["part"] = part;
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["inverse"] = inverse;
        ctx->saved_data["amplitude"] = amplitude;
        return rotary_out(q, or_none(k), {turns, positions, part, interleaved, inverse, amplitude});
    }
    // the inverse turn, itself differentiable
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        auto s = ctx->get_saved_variables();
        const int64_t part = ctx->saved_data["part"].toInt();
        const bool inter = ctx->saved_data["interleaved"].toBool(), inv = ctx->saved_data["inverse"].toBool();
        const double amp = ctx->saved_data["amplitude"].toDouble();
        const Tensor gk = g.size() > 1 ? g[1] : Tensor();
        variable_list d = wants_grad({&g[0], &gk}) ? RotaryFn::apply(g[0], maybe(gk), s[0], maybe(s[1]), part, inter, !inv, amp)
                                                   : rotary_out(g[0], gk, {s[0], s[1], part, inter, !inv, amp});
        Tensor none;
        return {d[0], d.size() > 1 ? d[1] : none, none, none, none, none, none, none};
    }
};

std::vector<Tensor> rotary(const Tensor &q, const std::optional<Tensor> &k_, const Tensor &turns, const std::optional<Tensor> &positions_,
                           int64_t part, bool interleaved, double amplitude) {
    const Tensor k = or_none(k_);
    const RotaryHow w{turns, or_none(positions_), part, interleaved, false, amplitude};
    rotary_check("rotary", q, k, w);
    return wants_grad({&q, &k}) ? RotaryFn::apply(q, k_, w.turns, positions_, part, interleaved, false, amplitude) : rotary_out(q, k, w);
}

// Whether an element of t lies `off` elements behind its first, the dimension `skip` aside: the largest strides first, which
// is exact for slices of one tensor (no inner part longer than an outer stride); what it finds is there in any case.
bool reaches(const Tensor &t, int64_t off, int64_t skip = -1) {
    std::vector<int64_t> dims;
    for (int64_t i = 0; i < t.dim(); ++i)
        if (i != skip && t.size(i) > 1 && t.stride(i) > 0) dims.push_back(i);
    std::sort(dims.begin(), dims.end(), [&](int64_t a, int64_t b) { return t.stride(a) > t.stride(b); });
    for (int64_t i : dims) off -= std::min(off / t.stride(i), t.size(i) - 1) * t.stride(i);
    return off == 0;
}
bool overlaps_itself(const Tensor &t) {
    if (at::has_internal_overlap(t) == at::MemOverlap::Yes) return true;
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1 && reaches(t, t.stride(i), i)) return true;
    return false;
}
bool overlap(const Tensor &a, const Tensor &b) {
    const auto s = at::get_overlap_status(a, b);
    if (s == at::MemOverlapStatus::Full || s == at::MemOverlapStatus::Partial) return true;
    if (s == at::MemOverlapStatus::No || !a.is_alias_of(b)) return false;
    const int64_t off = b.storage_offset() - a.storage_offset();
    return off < 0 ? reaches(b, -off) : reaches(a, off);
}

void rotary_inplace(const Tensor &q, const std::optional<Tensor> &k_, const Tensor &turns, const std::optional<Tensor> &positions_,
                    int64_t part, bool interleaved, double amplitude) {
    const Tensor k = or_none(k_);
    const RotaryHow w{turns, or_none(positions_), part, interleaved, false, amplitude};
    VALUE_CHECK(!wants_grad({&q, &k}), "rotary_: in place on a tensor that requires a gradient; use rotary()");
    auto check = [](const Tensor &t) {
        VALUE_CHECK(t.size(-1) == 1 || t.stride(-1) == 1, "rotary_: the elements of a head must lie side by side");
        VALUE_CHECK(!overlaps_itself(t), "rotary_: heads of one tensor share memory");
    };
    plain("rotary_", {&q, &k});
    VALUE_CHECK(q.dim() == 4, "rotary_: q must be [B, T, H, D], got ", q.sizes());
    check(q);
    if (k.defined()) {
        VALUE_CHECK(k.dim() == 4, "rotary_: k must be [B, T, Hk, D], got ", k.sizes());
        check(k);
        VALUE_CHECK(!overlap(q, k), "rotary_: q and k share memory");
    }
    rotary_check("rotary_", q, k, w);
    // first, as it refuses inference tensors outside inference mode
    q.unsafeGetTensorImpl()->bump_version();
    if (k.defined()) k.unsafeGetTensorImpl()->bump_version();
    if (q.numel() || (k.defined() && k.numel())) rotary_launch(q, k, q, k, w);
}

// --------------------------------------------------------- window attention

struct AttnHow {
    Tensor lengths;
    int64_t window, sinks;
    double scale;
};

int32_t clamped(int64_t x) { return (int32_t)std::min(x, (int64_t)1 << 30); }

void attention_check(const char *who, const Tensor &q, const Tensor &k, const Tensor &v, const AttnHow &w, bool decode) {
    plain(who, {&q, &k, &v, &w.lengths});
    if (decode) {
        VALUE_CHECK(q.dim() == 3, who, ": q must be [B, H, D], got ", q.sizes());
    } else {
        VALUE_CHECK(q.dim() == 4, who, ": q must be [B, T, H, D], got ", q.sizes());
    }
    const char *kv = decode ? ": k and v must be [B, T, Hkv, D]" : ": k and v must be [B, T, Hkv, D] with q's T";
    VALUE_CHECK(k.dim() == 4 && v.dim() == 4 && k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(3) == q.size(-1) &&
                          (decode || k.size(1) == q.size(1)),
                      who, kv, ", got ", k.sizes(), " and ", v.sizes(), " for q ", q.sizes());
    const int64_t H = q.size(-2), Hkv = k.size(2), D = q.size(-1);
    VALUE_CHECK(Hkv > 0 && H > 0 && H % Hkv == 0, who, ": ", H, " query heads do not share ", Hkv, " key heads evenly");
    VALUE_CHECK(D >= 1 && D <= 128, who, ": heads of 1 to 128 elements, got ", D);
    VALUE_CHECK(w.window >= 1, who, ": window must be at least 1, got ", w.window);
    VALUE_CHECK(w.sinks >= 0, who, ": sinks must not be negative, got ", w.sinks);
    VALUE_CHECK(std::isfinite((float)w.scale), who, ": scale must be finite");
    VALUE_CHECK(q.size(0) <= 65535 && H <= 65535, who, ": at most 65535 sequences and heads");
    VALUE_CHECK(k.size(1) <= (int64_t)1 << 30, who, ": at most 2^30 tokens");
    type_of(q, who, "q");
    TYPE_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), who, ": q, k and v differ in type");
    if (w.lengths.defined()) {
        TYPE_CHECK(w.lengths.scalar_type() == at::kInt, who, ": lengths must be int32");
        VALUE_CHECK(w.lengths.dim() == 1 && w.lengths.size(0) == q.size(0), who, ": lengths must be [B], got ", w.lengths.sizes());
    }
    same_device(who, q, {&k, &v, &w.lengths});
}

cail_ops_attention_args attention_args(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &o, const AttnHow &w) {
    cail_ops_attention_args a = {};
    a.type = type_of(q, "window_attention", "q");
    a.B = (int)q.size(0), a.T = (int)k.size(1), a.H = (int)q.size(-2), a.Hkv = (int)k.size(2), a.D = (int)q.size(-1);
    a.window = clamped(w.window), a.sinks = clamped(w.sinks);
    a.scale = (float)w.scale;
    a.lengths = w.lengths.defined() ? w.lengths.data_ptr<int32_t>() : nullptr;
    a.q = view(q), a.k = view(k), a.v = view(v), a.o = view(o);
    return a;
}

Tensor attention_forward(const Tensor &q, const Tensor &k, const Tensor &v, const AttnHow &w, float *lse, const Tensor &rest) {
    Tensor o = at::empty(q.sizes(), q.options());
    if (!o.numel()) return o;
    c10::cuda::CUDAGuard guard(q.device());
    cail_ops_attention_args a = attention_args(q, k, v, o, w);
    a.lse = lse;
    if (rest.defined()) a.o_rest = view(rest), a.rest_rows = (int)rest.size(1);
    done(L.attention(&a, stream_of(q)));
    return o;
}

struct AttentionFn : torch::autograd::Function<AttentionFn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &q_, const Tensor &k_, const Tensor &v_, const std::optional<Tensor> &lengths_,
                          int64_t window, int64_t sinks, double scale) {
        const Tensor lengths = or_none(lengths_);
        const Tensor q = rows(q_), k = rows(k_), v = rows(v_);
        Tensor lse = at::empty({(int64_t)CAIL_OPS_LSE_FLOATS(q.size(0), q.size(2), q.size(1))}, q.options().dtype(at::kFloat));
        const int64_t kept = cail_ops_rest_rows((int)q.size(1), (int)q.size(3), clamped(window), clamped(sinks));
        Tensor rest = q.scalar_type() == at::kFloat ? Tensor() : at::empty({q.size(0), kept, q.size(2), q.size(3)}, q.options());
        Tensor o = attention_forward(q, k, v, {lengths, window, sinks, scale}, lse.data_ptr<float>(), rest);
        ctx->save_for_backward({q, k, v, o, lse, lengths, rest});
        ctx->saved_data["window"] = window;
        ctx->saved_data["sinks"] = sinks;
        ctx->saved_data["scale"] = scale;
        return o;
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), "window_attention: the backward pass has no gradient of its own");
        auto s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2], &o = s[3], &lse = s[4];
        Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options());
        if (q.numel()) {
            c10::cuda::CUDAGuard guard(q.device());
            const Tensor dout = for_tiles(rows(g[0]));
            cail_ops_attention_args a = attention_args(q, k, v, o, {s[5], ctx->saved_data["window"].toInt(), ctx->saved_data["sinks"].toInt(),
                                                                   ctx->saved_data["scale"].toDouble()});
            a.dout = view(dout), a.dq = view(dq), a.dk = view(dk), a.dv = view(dv);
            a.lse = lse.data_ptr<float>();
            if (s[6].defined()) a.o_rest = view(s[6]), a.rest_rows = (int)s[6].size(1);
            Tensor delta = at::empty_like(lse);
            a.delta = delta.data_ptr<float>();
            a.workspace_bytes = L.workspace(&a);
            Tensor space;
            if (a.workspace_bytes) {
                space = at::empty({(int64_t)a.workspace_bytes}, q.options().dtype(at::kByte));
                a.workspace = space.data_ptr();
            }
            done(L.attention_backward(&a, stream_of(q)));
        }
        Tensor none;
        return {dq, dk, dv, none, none, none, none};
    }
};

Tensor window_attention_on(const Tensor &q_, const Tensor &k_, const Tensor &v_, const AttnHow &w) {
    const Tensor q = for_tiles(q_), k = for_tiles(k_), v = for_tiles(v_);
    if (wants_grad({&q, &k, &v})) return AttentionFn::apply(q, k, v, maybe(w.lengths), w.window, w.sinks, w.scale);
    return attention_forward(rows(q), rows(k), rows(v), w, nullptr, Tensor());
}

Tensor window_attention(const Tensor &q, const Tensor &k, const Tensor &v, int64_t window, int64_t sinks, const std::optional<Tensor> &lengths_,
                        const std::optional<double> &scale_) {
    AttnHow w{or_none(lengths_), window, sinks, 0.0};
    w.scale = scale_.has_value() ? *scale_ : q.dim() > 0 && q.size(-1) > 0 ? 1.0 / std::sqrt((double)q.size(-1)) : 1.0;
    attention_check("window_attention", q, k, v, w, false);
    if (w.lengths.defined()) w.lengths = w.lengths.contiguous();
    const int64_t D = q.size(3);
    if (D % 8 && q.scalar_type() != at::kFloat && q.size(1) > kCopyFrom && q.numel()) {
        // heads of a size that the tile loads do not take, as the next size that they do: zeros add nothing to a product
        auto padded = [&](const Tensor &t) { return at::constant_pad_nd(t, {0, 8 - D % 8}); };
        return window_attention_on(padded(q), padded(k), padded(v), w).narrow(3, 0, D).contiguous();
    }
    return window_attention_on(q, k, v, w);
}

Tensor window_attention_decode(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &lengths, int64_t window, int64_t sinks,
                               const std::optional<double> &scale_) {
    AttnHow w{lengths, window, sinks, 0.0};
    w.scale = scale_.has_value() ? *scale_ : q.dim() > 0 && q.size(-1) > 0 ? 1.0 / std::sqrt((double)q.size(-1)) : 1.0;
    VALUE_CHECK(!wants_grad({&q, &k, &v}), "window_attention_decode: has no backward pass; call it under torch.no_grad()");
    attention_check("window_attention_decode", q, k, v, w, true);
    for (const Tensor *c : {&k, &v})
        VALUE_CHECK(c->size(-1) == 1 || c->stride(-1) == 1, "window_attention_decode: the elements of a cached head must lie side by side");
    w.lengths = w.lengths.contiguous();
    const Tensor qr = rows(q);
    Tensor o = at::empty(q.sizes(), q.options());
    if (!o.numel()) return o;
    c10::cuda::CUDAGuard guard(q.device());
    const cail_ops_attention_args a = attention_args(qr, k, v, o, w);
    done(L.decode(&a, stream_of(q)));
    return o;
}

// ------------------------------------------------------------- distillation

constexpr int64_t kStats = 8;

cail_ops_distill_args distill_args(const Tensor &z, const Tensor &ids, const Tensor &t, const Tensor &y, double tau, double hard, int64_t mean) {
    cail_ops_distill_args a = {};
    a.type = type_of(z, "distill_loss", "logits");
    a.N = z.size(0), a.V = z.size(1), a.K = (int)ids.size(1);
    a.logits = z.data_ptr(), a.ld_logits = z.stride(0);
    a.ids = ids.data_ptr(), a.ids64 = ids.scalar_type() == at::kLong;
    a.teacher = t.data_ptr(), a.teacher_type = type_of(t, "distill_loss", "teacher_logits");
    a.targets = y.defined() ? y.data_ptr<int64_t>() : nullptr;
    a.temperature = (float)tau, a.hard_weight = (float)hard, a.mean = (int)mean;
    return a;
}

// the row losses, what backward needs of a row, and the factor, in one buffer
struct DistillKept {
    Tensor buffer;
    float *rows, *stats, *factor;
    DistillKept(Tensor b, int64_t N) : buffer(std::move(b)) {
        float *p = buffer.data_ptr<float>();
        stats = p, factor = p + N * kStats, rows = p + N * kStats + 1;
    }
};

Tensor distill_forward(const Tensor &z, const Tensor &ids, const Tensor &t, const Tensor &y, double tau, double hard, int64_t mean, Tensor *kept) {
    const int64_t N = z.size(0);
    c10::cuda::CUDAGuard guard(z.device());
    const auto f32 = z.options().dtype(at::kFloat);
    Tensor loss = mean == -1 ? at::empty({N}, f32) : at::empty({}, f32);
    DistillKept w(at::empty({N * (kStats + 1) + 1}, f32), N);
    cail_ops_distill_args a = distill_args(z, ids, t, y, tau, hard, mean);
    a.stats = w.stats, a.factor = w.factor;
    a.rows = mean == -1 ? loss.data_ptr<float>() : w.rows;
    a.loss = mean == -1 ? nullptr : loss.data_ptr<float>();
    done(L.distill(&a, stream_of(z)));
    if (kept) *kept = w.buffer;
    return loss;
}

struct DistillFn : torch::autograd::Function<DistillFn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &z, const Tensor &ids, const Tensor &t, const std::optional<Tensor> &y_, double tau,
                          double hard, int64_t mean) {
        const Tensor y = or_none(y_);
        Tensor kept, loss = distill_forward(z, ids, t, y, tau, hard, mean, &kept);
        ctx->save_for_backward({z, ids, t, y, kept});
        ctx->saved_data["tau"] = tau;
        ctx->saved_data["hard"] = hard;
        ctx->saved_data["mean"] = mean;
        return loss;
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), "distill_loss: the backward pass has no gradient of its own");
        auto s = ctx->get_saved_variables();
        const Tensor &z = s[0];
        const int64_t N = z.size(0), V = z.size(1), ld = z.stride(0);
        // the gradient's rows lie as the logits' rows do, where that costs
        // little, so that both are on the same offsets from 16 bytes
        Tensor dz = N > 1 && ld > V && ld < 2 * V ? at::empty_strided({N, V}, {ld, 1}, z.options()) : at::empty({N, V}, z.options());
        if (N) {
            c10::cuda::CUDAGuard guard(z.device());
            const Tensor gl = g[0].to(at::kFloat).contiguous();
            const int64_t mean = ctx->saved_data["mean"].toInt();
            cail_ops_distill_args a = distill_args(z, s[1], s[2], s[3], ctx->saved_data["tau"].toDouble(), ctx->saved_data["hard"].toDouble(), mean);
            DistillKept w(s[4], N);
            a.stats = w.stats, a.factor = w.factor;
            a.grad_loss = gl.data_ptr<float>();
            a.grad = dz.data_ptr(), a.ld_grad = N > 1 ? dz.stride(0) : V;
            done(L.distill_backward(&a, stream_of(z)));
        }
        Tensor none;
        return {dz, none, none, none, none, none, none};
    }
};

Tensor distill_loss(const Tensor &z_, const Tensor &ids_, const Tensor &t_, const std::optional<Tensor> &y_, double tau, double hard, int64_t mean) {
    const char *who = "distill_loss";
    Tensor y = or_none(y_);
    plain(who, {&z_, &ids_, &t_, &y});
    VALUE_CHECK(z_.dim() == 2 && z_.size(1) > 0, who, ": logits must be [N, V], got ", z_.sizes());
    VALUE_CHECK(z_.size(1) <= kIntMax, who, ": at most 2^31 - 1 logits in a row");
    VALUE_CHECK(ids_.dim() == 2 && ids_.size(0) == z_.size(0) && t_.sizes() == ids_.sizes(), who,
                      ": teacher_ids and teacher_logits must be [N, K] with the logits' N, got ", ids_.sizes(), " and ", t_.sizes());
    VALUE_CHECK(ids_.size(1) <= CAIL_OPS_DISTILL_MAX_K, who, ": at most ", CAIL_OPS_DISTILL_MAX_K, " teacher entries in a row, got ", ids_.size(1));
    type_of(z_, who, "logits");
    type_of(t_, who, "teacher_logits");
    TYPE_CHECK(ids_.scalar_type() == at::kLong || ids_.scalar_type() == at::kInt, who, ": teacher_ids must be int32 or int64");
    if (y.defined()) {
        VALUE_CHECK(y.dim() == 1 && y.size(0) == z_.size(0), who, ": targets must be [N], got ", y.sizes());
        TYPE_CHECK(y.scalar_type() == at::kLong || y.scalar_type() == at::kInt, who, ": targets must be int32 or int64");
    }
    VALUE_CHECK(std::isfinite(tau) && tau > 0 && (float)tau > 0 && std::isfinite(1.f / (float)tau), who, ": temperature must be positive, got ", tau);
    VALUE_CHECK(hard >= 0 && hard <= 1, who, ": hard_weight must be in [0, 1], got ", hard);
    VALUE_CHECK(hard == 0 || y.defined(), who, ": hard_weight needs targets");
    VALUE_CHECK(!wants_grad({&t_}), who, ": the teacher's logits get no gradient; detach them");
    same_device(who, z_, {&ids_, &t_, &y});
    // rows side by side, or further apart; a copy where they are not
    const Tensor z = z_.size(1) == 1 || z_.stride(1) == 1 ? (z_.size(0) <= 1 || z_.stride(0) >= z_.size(1) ? z_ : z_.contiguous()) : z_.contiguous();
    const Tensor ids = ids_.contiguous(), t = t_.contiguous();
    if (y.defined()) y = y.to(at::kLong).contiguous();
    if (wants_grad({&z})) return DistillFn::apply(z, ids, t, maybe(y), tau, hard, mean);
    return distill_forward(z, ids, t, y, tau, hard, mean, nullptr);
}

int64_t launches() { return (int64_t)L.launches(); }

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "window attention, rotary positions and distillation on tensors through libcail_ops.so";
    m.def("load", &load, "open libcail_ops.so");
    m.def("rotary", &rotary);
    m.def("rotary_inplace", &rotary_inplace);
    m.def("window_attention", &window_attention);
    m.def("window_attention_decode", &window_attention_decode);
    m.def("distill_loss", &distill_loss);
    m.def("launches", &launches);
}
