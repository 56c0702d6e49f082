"""Window attention, rotary positions and distillation against plain 64-bit
forms (tests/lm_reference.py), and their refusals.

Tolerances, as 2-norms relative to the wanted result.  u is half a step of
the type (bf16 2^-8 ... as torch.finfo(t).eps / 2), e = 2^-24 that of float32.

* Rotary: one rounding of each output (u) after two products and a sum in 32
  bits of a sine and cosine good to 4 e: at most u + 8 e.
* Attention forward: the output's rounding (u), and the probabilities'
  rounding to the type before the second product (at most u relative to each
  term).  Terms of either sign: the error's 2-norm is at most u times the norm
  of p |v|, which for values of independent sign is of the order of the
  output's own norm; 32-bit sums add e times the number of terms' root.  Bound
  used: 3 u + 64 e (64 e: scores of up to |s| = 32 carry s e each in the
  exponent, and sums of up to a few hundred terms).
* Attention gradients: the same two roundings, and ds = p (dp - delta) is
  rounded where it enters a product, where dp - delta cancels partly (the
  norm of ds is kept by its terms, so u stays relative to them): 5 u + 256 e.
* Distillation: loss in 32 bits, of at most 16 e |z| / tau for the exponents
  and 8 e for sums and logarithms: 2e-6 on losses of the order of 1 to 10.
  Gradient: one rounding u, and 64 e from exponents of up to 32.
"""
import random
import threading

import pytest
import torch

import lm_reference as ref

TYPES = [torch.float32, torch.bfloat16, torch.float16]
E = 2.0 ** -24


def ids_of(t):
    return str(t).replace("torch.", "")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, by=1.0):
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * by).to(dtype).cuda()


def ops():
    from cail_b200 import ops as o

    return o


@pytest.fixture(scope="module", autouse=True)
def built(build):
    from cail_b200.ops import ext

    ext.build_ops()


# ------------------------------------------------------------ refusals (CPU)


def test_rotary_plan_refuses():
    R = ops().Rotary
    for kw in (dict(dim=3), dict(dim=0), dict(dim=64, base=0.0), dict(dim=64, factor=0.0), dict(dim=64, scaling="other"),
               dict(dim=2, scaling="ntk", factor=2.0), dict(dim=64, scaling="parts", factor=2.0),
               dict(dim=64, scaling="parts", factor=2.0, original=8, fast=1.0, slow=1.0)):
        with pytest.raises(ValueError):
            R(device="cpu", **kw)


def test_rotary_refuses():
    o = ops()
    plan = o.Rotary(8, device="cpu")
    q = torch.zeros(2, 3, 4, 8)
    bad = [
        (ValueError, (q[0], None)), (ValueError, (torch.zeros(2, 3, 4, 6), None)), (ValueError, (q, torch.zeros(2, 2, 4, 8))),
        (TypeError, (q, q.half())), (TypeError, (q.double(), None)), (ValueError, (q, None, torch.zeros(2, dtype=torch.int64))),
        (TypeError, (q, None, torch.zeros(3))), (ValueError, (q, None, torch.zeros(2, 4, dtype=torch.int32))),
        (ValueError, (torch.zeros(1, 1, 1, 1026), None)),
    ]
    for kind, args in bad:
        with pytest.raises(kind):
            o.rotary(args[0], args[1], plan, *args[2:])
        with pytest.raises(kind):
            o.rotary_(args[0], args[1], plan, *args[2:])
    with pytest.raises(ValueError, match="CUDA"):
        o.rotary(q, None, plan)
    with pytest.raises(ValueError, match="gradient"):
        o.rotary_(q.clone().requires_grad_(), None, plan)
    with pytest.raises(ValueError, match="share memory"):
        o.rotary_(q, q, plan)
    with pytest.raises(ValueError, match="share memory"):
        o.rotary_(torch.zeros(1, 3, 4, 8).expand(2, 3, 4, 8), None, plan)
    with pytest.raises(ValueError, match="side by side"):
        o.rotary_(torch.zeros(2, 3, 8, 4).transpose(2, 3), None, plan)


def test_rotary_in_place_refuses_slices_that_overlap():
    """Slices of one projection: what overlaps is refused, what does not goes on (to the next check: the device)."""
    o = ops()
    plan = o.Rotary(8, device="cpu")
    x = torch.zeros(2, 3, 6, 8)
    wide = torch.zeros(2, 3, 2, 20)
    for q, k in ((x[:, :, :4], x[:, :, :4]), (x[:, :, :4], x[:, :, 2:6]), (x[:, :, 2:6], x[:, :, 1:3]), (x[:, :, ::2], x[:, :, :3]),
                 (wide[..., :8], wide[..., 7:15]), (wide[..., 4:12], wide[..., :8]), (x[:, :, 5:], x[:, :, 3:])):
        with pytest.raises(ValueError, match="share memory"):
            o.rotary_(q, k, plan)
    for t in (torch.zeros(100).as_strided((1, 6, 1, 8), (1, 4, 1, 1)), torch.zeros(400).as_strided((2, 3, 2, 8), (8, 16, 8, 1))):
        with pytest.raises(ValueError, match="share memory"):
            o.rotary_(t, None, plan)
    flat = torch.zeros(2, 3, 6 * 8)
    views = [z.view(2, 3, 2, 8) for z in flat.split(16, dim=2)]
    for q, k in ((x[:, :, :4], x[:, :, 4:]), (x[:, :, ::2], x[:, :, 1::2]), (wide[..., :8], wide[..., 8:16]), (views[0], views[1]),
                 (views[2], views[0]), (x[:1], x[1:]), (x[:, :1], x[:, 1:2]), (x[:, :, :0], x), (x.transpose(0, 1), None),
                 (torch.zeros(2, 3, 1, 8)[:, :, :1], None), (torch.zeros(1, 1, 1, 8), None)):
        with pytest.raises(ValueError, match="CUDA"):
            o.rotary_(q, k, plan)


def test_window_attention_refuses():
    o = ops()
    q, k = torch.zeros(2, 5, 4, 8), torch.zeros(2, 5, 2, 8)
    n = torch.zeros(2, dtype=torch.int32)
    bad = [
        (ValueError, (q[0], k, k, 4)), (ValueError, (q, k[:, :4], k[:, :4], 4)), (ValueError, (q, k, k[:, :, :1], 4)),
        (ValueError, (q, torch.zeros(2, 5, 3, 8), torch.zeros(2, 5, 3, 8), 4)), (ValueError, (q, k[:, :, :0], k[:, :, :0], 4)),
        (ValueError, (torch.zeros(2, 5, 4, 136), torch.zeros(2, 5, 2, 136), torch.zeros(2, 5, 2, 136), 4)),
        (ValueError, (q, k, k, 0)), (ValueError, (q, k, k, -1)), (ValueError, (q, k, k, 4, -1)),
        (TypeError, (q, k.half(), k, 4)), (TypeError, (q.double(), k.double(), k.double(), 4)),
        (TypeError, (q, k, k, 4, 0, n.long())), (ValueError, (q, k, k, 4, 0, n[:1])),
        (ValueError, (q, k, k, 4, 0, None, float("nan"))), (ValueError, (q, k, k, 4)),
    ]
    for kind, args in bad:
        with pytest.raises(kind):
            o.window_attention(*args)
    with pytest.raises(ValueError, match="CUDA"):
        o.window_attention(q, k, k, 4)
    one = torch.zeros(2, 4, 8)
    for kind, args in [
        (ValueError, (q, k, k, n, 4)), (ValueError, (one, k, k[:1], n, 4)), (TypeError, (one, k, k, n.long(), 4)),
        (ValueError, (one, k, k, n, 0)), (ValueError, (one.clone().requires_grad_(), k, k, n, 4)), (ValueError, (one, k, k, n, 4)),
    ]:
        with pytest.raises(kind):
            o.window_attention_decode(*args)


def test_distill_loss_refuses():
    o = ops()
    z, ids, t, y = torch.zeros(3, 11), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2), torch.zeros(3, dtype=torch.int64)
    bad = [
        (ValueError, dict(logits=z[0])), (ValueError, dict(teacher_ids=ids[:2])), (ValueError, dict(teacher_logits=t[:, :1])),
        (TypeError, dict(teacher_ids=t)), (TypeError, dict(logits=z.double())), (TypeError, dict(teacher_logits=t.double())),
        (ValueError, dict(targets=y[:2])), (TypeError, dict(targets=y.float())), (ValueError, dict(temperature=0.0)),
        (ValueError, dict(temperature=float("inf"))), (ValueError, dict(temperature=1e-45)), (ValueError, dict(hard_weight=1.5)),
        (ValueError, dict(hard_weight=0.5)), (ValueError, dict(reduction="median")),
        (ValueError, dict(teacher_logits=t.clone().requires_grad_())),
        (ValueError, dict(teacher_ids=torch.zeros(3, 1025, dtype=torch.int64), teacher_logits=torch.zeros(3, 1025))),
        (ValueError, dict(logits=torch.zeros(3, 0))),
    ]
    for kind, kw in bad:
        with pytest.raises(kind):
            o.distill_loss(**{**dict(logits=z, teacher_ids=ids, teacher_logits=t), **kw})
    with pytest.raises(ValueError, match="CUDA"):
        o.distill_loss(z, ids, t)


def test_tensors_that_a_pointer_does_not_show_are_refused():
    """A negation still to be done, a forward-mode tangent, a sparse layout, sizes past 32 bits."""
    import torch.autograd.forward_ad as fwd
    o = ops()
    plan = o.Rotary(8, device="cpu")
    q, z = torch.zeros(2, 5, 2, 8), torch.zeros(3, 11)
    n = torch.zeros(2, dtype=torch.int32)
    ids, t = torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2)

    def calls(q, z):
        return [lambda: o.rotary(q, None, plan), lambda: o.rotary_(q, None, plan), lambda: o.window_attention(q, q, q, 4),
                lambda: o.window_attention_decode(q[:, 0], q, q, n, 4), lambda: o.distill_loss(z, ids, t)]

    negated = [torch.zeros(x.shape, dtype=torch.complex64).conj().imag for x in (q, z)]
    assert negated[0].is_neg()
    for call in calls(*negated):
        with pytest.raises(ValueError, match="negation"):
            call()
    for call in calls(q.to_sparse(), z.to_sparse()):
        with pytest.raises((ValueError, RuntimeError)):
            call()
    with fwd.dual_level():
        for call in calls(*(fwd.make_dual(x, torch.ones_like(x)) for x in (q, z))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
    for shape in ((1, 2 ** 32 + 5, 1, 8), (2 ** 32 + 1, 1, 1, 8), (1, 1, 2 ** 32 + 1, 8)):
        with pytest.raises(ValueError, match="at most"):
            o.rotary(torch.zeros(1).expand(shape), None, plan)
        with pytest.raises(ValueError, match="at most"):
            o.window_attention(*[torch.zeros(1).expand(shape)] * 3, 4)
    with pytest.raises(ValueError, match="scale"):
        o.window_attention(q, q, q, 4, scale=1e300)


def test_c_entries_refuse_without_touching_a_device():
    """Bad sizes come back as CAIL_OPS_EINVAL with a text, before any CUDA call."""
    import ctypes
    import os

    from conftest import LIB

    lib = ctypes.CDLL(os.path.join(LIB, "libcail_ops.so"))
    lib.cail_ops_last_error.restype = ctypes.c_char_p
    zero = (ctypes.c_char * 1024)()
    for name in ("cail_ops_window_attention", "cail_ops_window_attention_backward", "cail_ops_window_attention_decode",
                 "cail_ops_distill", "cail_ops_distill_backward", "cail_ops_rotary"):
        assert getattr(lib, name)(ctypes.byref(zero), None) == 1, name
        assert lib.cail_ops_last_error() != b""


def attention_args(T, window, sinks, dtype, B=1, H=1, Hkv=1, D=64):
    """cail_ops_attention_args of contiguous arrays at made-up addresses, for questions that touch no device."""
    import ctypes as c

    class Bthd(c.Structure):
        _fields_ = [("ptr", c.c_void_p), ("sb", c.c_int64), ("st", c.c_int64), ("sh", c.c_int64)]

    class Args(c.Structure):
        _fields_ = ([(n, c.c_int) for n in ("type", "B", "T", "H", "Hkv", "D", "window", "sinks")] + [("scale", c.c_float), ("lengths", c.c_void_p)] +
                    [(n, Bthd) for n in "qkvo"] + [("lse", c.c_void_p), ("o_rest", Bthd), ("rest_rows", c.c_int)] +
                    [(n, Bthd) for n in ("dout", "dq", "dk", "dv")] + [("delta", c.c_void_p), ("workspace", c.c_void_p), ("workspace_bytes", c.c_size_t)])

    a = Args(TYPES.index(dtype), B, T, H, Hkv, D, window, sinks, 0.125, None)
    at = lambda h, n=T: Bthd(1 << 20, n * h * D, h * D, D)  # noqa: E731
    a.q = a.o = a.dout = a.dq = at(H)
    a.k = a.v = a.dk = a.dv = at(Hkv)
    a.lse = a.delta = 1 << 20
    a.rest_rows = min(T, 128)
    a.o_rest = at(H, a.rest_rows)
    return a


@pytest.mark.parametrize("dtype", TYPES[1:], ids=ids_of)
@pytest.mark.parametrize("T", [65533 * 128, 65534 * 128, 65534 * 128 + 1, 65535 * 128])
@pytest.mark.parametrize("sinks", [4, 128, 129, 1000])
def test_parts_of_the_sinks_stay_inside_a_grid(dtype, T, sinks):
    """The tensor-core kernels' grid has one block in z for every tile of 128 keys, and more where the sinks' tiles are cut into
    parts (as many as the workspace has room for): at most 65535 in all."""
    import ctypes
    import os

    from conftest import LIB

    lib = ctypes.CDLL(os.path.join(LIB, "libcail_ops.so"))
    lib.cail_ops_window_attention_workspace.restype = ctypes.c_size_t
    room = [lib.cail_ops_window_attention_workspace(ctypes.byref(attention_args(T, 20, n, dtype))) for n in (sinks, 0)]
    tiles, sunk, part = (T + 127) // 128, (sinks + 127) // 128, 2 * 128 * 64 * 4
    assert (room[0] - room[1]) % (sunk * part) == 0
    parts = (room[0] - room[1]) // (sunk * part)
    assert tiles + sunk * max(parts - 1, 0) <= 65535


def test_a_workspace_can_be_asked_for_without_a_device():
    """In a process of its own: a division by the number of a missing device's SMs would end it."""
    import os
    import subprocess
    import sys

    code = ("import ctypes, sys; sys.path[:0] = ['tests', '.']; import torch, test_lm_ops as t; from conftest import LIB\n"
            "lib = ctypes.CDLL(LIB + '/libcail_ops.so'); f = lib.cail_ops_window_attention_workspace; f.restype = ctypes.c_size_t\n"
            "print([f(ctypes.byref(t.attention_args(T, 20, 4, d))) for d in t.TYPES for T in (500, 100000)])")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       env={**os.environ, "CUDA_VISIBLE_DEVICES": ""})
    assert r.returncode == 0, r.stderr[-500:]
    assert all(n > 0 for n in eval(r.stdout.splitlines()[-1])[1::2])


# -------------------------------------------------------------------- rotary

SCALINGS = [dict(), dict(scaling="linear", factor=8.0), dict(scaling="ntk", factor=4.0), dict(scaling="parts", factor=16.0, original=2048)]


def freqs(dim, base=10000.0, scaling=None, factor=1.0, original=0, fast=32.0, slow=1.0):
    import math

    if scaling == "ntk":
        base *= factor ** (dim / (dim - 2))
    f = [base ** (-2 * i / dim) for i in range(dim // 2)]
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling == "parts":
        out = []
        for x in f:
            turns = original * x / (2 * math.pi)
            w = min(1.0, max(0.0, (turns - slow) / (fast - slow)))
            out.append(x * w + x / factor * (1 - w))
        f = out
    return f, (0.1 * math.log(factor) + 1 if scaling == "parts" else 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("inter", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("B,T,H,Hk,D,part", [(1, 1, 1, 1, 2, 2), (2, 7, 3, 1, 64, 64), (3, 130, 4, 2, 80, 20), (1, 33, 2, 2, 128, 64),
                                             (2, 5, 5, 3, 17, 6), (1, 3, 40, 8, 1024, 1024), (2, 1, 7, 7, 40, 38)])
def test_rotary_matches_64_bit(dtype, inter, B, T, H, Hk, D, part):
    o = ops()
    g = gen(B * 100 + D)
    for n, how in enumerate(SCALINGS):
        if how.get("scaling") == "ntk" and part < 4:
            continue
        plan = o.Rotary(part, interleaved=inter, **how)
        f, amp = freqs(part, **how)
        q, k = randn(g, B, T, H, D, dtype=dtype), randn(g, B, T, Hk, D, dtype=dtype)
        pos = [None, torch.randint(0, 10 ** 6, (T,), generator=g).cuda(), torch.randint(-50, 300000, (B, T), generator=g).int().cuda(),
               torch.arange(T).cuda() + 2 ** 31][n]
        at = torch.arange(T).cuda() if pos is None else pos
        at = at.expand(B, T) if at.dim() == 1 else at
        q.requires_grad_(), k.requires_grad_()
        qo, ko = o.rotary(q, k, plan, pos)
        gq, gk = randn(g, B, T, H, D, dtype=dtype), randn(g, B, T, Hk, D, dtype=dtype)
        dq, dk = torch.autograd.grad((qo, ko), (q, k), (gq, gk))
        tol = ref.half_step(dtype) + 8 * E
        for got, x, inv in ((qo, q, False), (ko, k, False), (dq, gq, True), (dk, gk, True)):
            want = ref.rotate(x.detach(), at, f, amp, inter, inv)
            assert got.dtype == dtype and got.is_contiguous()
            assert ref.rel(got, want) <= tol, (how, inv)
        with torch.no_grad():
            q2, k2 = q.detach().clone(), k.detach().clone()
            a, b = o.rotary_(q2, k2, plan, pos)
            assert a is q2 and torch.equal(q2, qo) and torch.equal(k2, ko)
            assert torch.equal(o.rotary(q2, None, plan, pos), o.rotary(q2, k2, plan, pos)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("inter", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("first", [0, 100000, 2 ** 30])
def test_rotary_angles_lose_nothing(inter, first):
    """The pair (1, 0) turns into cosine and sine themselves: sincospif is good to one unit in the last place, E below 1, and what
    is left of the angle is put in with one more rounding, E / 2: 1.5 E in all (1.6 for the second order).  An angle rounded to
    32 bits would be off by up to pi / 2 E by itself."""
    o = ops()
    plan = o.Rotary(64, interleaved=inter)
    ia = torch.arange(0, 64, 2) if inter else torch.arange(32)
    ib = ia + (1 if inter else 32)
    q = torch.zeros(1, 5000, 1, 64, device="cuda")
    q[..., ia] = 1.0
    pos = (torch.arange(5000) + first).cuda()
    got = o.rotary(q, None, plan, pos)[0, :, 0].double()
    turns = pos.double()[:, None] * plan.turns
    angle = (turns - turns.round()) * 2 * torch.pi
    assert float((got[:, ia] - angle.cos()).abs().max()) <= 1.6 * E
    assert float((got[:, ib] - angle.sin()).abs().max()) <= 1.6 * E


@pytest.mark.gpu
@pytest.mark.parametrize("inter", [False, True], ids=["half", "interleaved"])
def test_rotary_strides(inter):
    """q and k as parts of one projection, heads before tokens, elements apart,
    rows on odd addresses, expanded gradients."""
    o = ops()
    g = gen(5)
    plan = o.Rotary(16, interleaved=inter)
    f, amp = freqs(16)
    at = torch.arange(6).cuda().expand(2, 6)
    tol = ref.half_step(torch.bfloat16) + 8 * E
    fused = randn(g, 2, 6, 3 * 4 * 20, dtype=torch.bfloat16)
    q, k = (x.view(2, 6, 4, 20) for x in fused.split(80, 2)[:2])
    flat = randn(g, 2 * 6 * 4 * 20 + 1, dtype=torch.bfloat16)
    odd = flat[1:].view(2, 6, 4, 20)
    for x in (q, k, q.transpose(1, 2).contiguous().transpose(1, 2), odd, randn(g, 2, 6, 20, 4, dtype=torch.bfloat16).transpose(2, 3),
              randn(g, 2, 6, 1, 20, dtype=torch.bfloat16).expand(2, 6, 4, 20)):
        assert ref.rel(o.rotary(x, None, plan), ref.rotate(x, at, f, amp, inter)) <= tol
    want = ref.rotate(q, at, f, amp, inter), ref.rotate(k, at, f, amp, inter)
    rest = fused[:, :, 160:].clone()
    o.rotary_(q, k, plan)  # in place on parts of one tensor; the rest of it stays
    assert ref.rel(q, want[0]) <= tol and ref.rel(k, want[1]) <= tol and torch.equal(fused[:, :, 160:], rest)
    x = randn(g, 2, 6, 4, 20).requires_grad_()
    o.rotary(x, None, plan).sum().backward()
    assert ref.rel(x.grad, ref.rotate(torch.ones_like(x), at, f, amp, inter, True)) <= 16 * E


@pytest.mark.gpu
def test_rotary_empty_and_second_derivative():
    o = ops()
    plan = o.Rotary(4)
    assert o.rotary(torch.zeros(0, 3, 2, 4).cuda(), torch.zeros(0, 3, 1, 4).cuda(), plan)[0].shape == (0, 3, 2, 4)
    assert o.rotary(torch.zeros(2, 0, 2, 4).cuda(), None, plan).shape == (2, 0, 2, 4)
    x = randn(gen(1), 1, 3, 2, 6).requires_grad_()
    y = o.rotary(x, None, plan)
    (d,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)  # 2 x on the rotation: turned there and back
    (dd,) = torch.autograd.grad(d.sum(), x)
    assert ref.rel(dd, torch.full_like(x, 2.0)) <= 32 * E


# ----------------------------------------------------------------- attention

# B, T, H, Hkv, D, window, sinks, lengths
ATTENTION = [
    (1, 1, 1, 1, 64, 1, 0, None),
    (2, 5, 2, 1, 16, 2, 1, [5, 0]),
    (1, 63, 2, 2, 33, 7, 3, None),
    (2, 64, 2, 1, 64, 64, 0, [64, 1]),
    (1, 65, 3, 3, 80, 1, 0, None),
    (1, 128, 2, 2, 128, 200, 5, None),
    (2, 129, 4, 2, 64, 33, 70, [129, 65]),
    (1, 200, 4, 1, 128, 64, 0, None),
    (3, 257, 2, 2, 72, 100, 130, [257, 128, 129]),
    (1, 511, 8, 2, 64, 128, 4, [500]),
    (1, 700, 2, 1, 128, 1000, 0, [699]),
    (2, 640, 2, 2, 8, 250, 1000, [640, 3]),
    (1, 1100, 1, 1, 64, 300, 260, None),
    (1, 1500, 4, 1, 128, 100, 3, [1400]),
    (2, 1025, 2, 1, 64, 64, 129, [1025, 200]),
    (1, 300, 2, 1, 100, 50, 2, [290]),
    (2, 190, 2, 2, 1, 30, 2, None),
    (1, 150, 3, 1, 127, 400, 0, None),
]


def attention_inputs(case, dtype, seed=0, by=1.0):
    B, T, H, Hkv, D, window, sinks, lengths = case
    g = gen(seed + T)
    q, k, v, do = (randn(g, B, T, h, D, dtype=dtype, by=by) for h in (H, Hkv, Hkv, H))
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32).cuda()
    return q, k, v, do, n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("case", ATTENTION, ids=str)
def test_window_attention_matches_64_bit(dtype, case):
    o = ops()
    window, sinks = case[5:7]
    q, k, v, do, n = attention_inputs(case, dtype)
    with torch.no_grad():
        plain = o.window_attention(q, k, v, window, sinks, lengths=n)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    out = o.window_attention(*leaves, window, sinks, lengths=n)
    assert torch.equal(out, plain)
    grads = torch.autograd.grad(out, leaves, do)
    r = [x.double().requires_grad_() for x in (q, k, v)]
    want = ref.attention(*r, window, sinks, n)
    dwant = torch.autograd.grad(want, r, do.double())
    u = ref.half_step(dtype)
    assert out.dtype == dtype and out.is_contiguous()
    assert ref.rel(out, want) <= 3 * u + 64 * E
    for name, got, w in zip("qkv", grads, dwant):
        assert got.dtype == dtype
        assert ref.rel(got, w) <= 5 * u + 256 * E, "d" + name
    if n is not None:  # rows behind a sequence: exact zeros
        for b, m in enumerate(n.tolist()):
            for x in (out, *grads):
                assert not x[b, m:].any()
    again = torch.autograd.grad(o.window_attention(*leaves, window, sinks, lengths=n), leaves, do)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES[1:], ids=ids_of)
@pytest.mark.parametrize("window, sinks, D", [(2, 0, 64), (3, 1, 128), (5, 4, 72), (200, 0, 16)])
def test_rows_of_few_keys_lose_one_rounding(dtype, window, sinks, D):
    """Element by element: o is off by its own rounding, dq and dk by their own and that of ds.  With u half a step, p and o
    reach delta = do.o to 2 u^2 and u^2 relative to their terms, so ds_ij to p_ij (A_ij + sum_j p_ij A_ij) 4 u^2 with
    A_ij = sum_d |do_id v_jd| (4 covers both ends of ds' own rounding); 256 E stands for the 32-bit sums of at most 128 terms
    and the exponentials; 16 E max|do| for ds that are tiny beside max|do|.  One more rounding of p or o in delta would be off
    by u times the same terms, 2^6 and more over this."""
    o = ops()
    T, H = 300, 2
    q, k, v, do, _ = attention_inputs((1, T, H, H, D, window, sinks, None), dtype)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    out = o.window_attention(*leaves, window, sinks)
    got = torch.autograd.grad(out, leaves, do)
    u, scale = ref.half_step(dtype), D ** -0.5
    on = ref.seen_mask(T, T, window, sinks, q.device)
    rows = 128 if window > 128 else T  # of few keys
    for h in range(H):
        qh, kh, vh, gh = (x[0, :, h].double() for x in (q, k, v, do))
        p = torch.softmax(torch.where(on, scale * qh @ kh.T, -1e300), -1) * on
        dp, A = gh @ vh.T, gh.abs() @ vh.abs().T
        ds = p * (dp - (p * dp).sum(-1, keepdim=True))
        off = p * (A + (p * A).sum(-1, keepdim=True)) * (4 * u * u + 256 * E) + on * 16 * E * float(gh.abs().max()) + u * ds.abs()
        want = p @ vh
        assert ((out[0, :, h].double() - want).abs() <= u * want.abs() + (2 * u * u + 256 * E) * (p @ vh.abs()))[:rows].all()
        want = scale * ds @ kh
        assert ((got[0][0, :, h].double() - want).abs() <= u * want.abs() + 1.01 * scale * off @ kh.abs())[:rows].all()
        want = scale * ds.T @ qh
        if rows == T:
            assert ((got[1][0, :, h].double() - want).abs() <= u * want.abs() + 1.01 * scale * off.T @ qh.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("what", [float("inf"), float("nan")])
def test_a_gradient_that_is_not_finite_stays_with_its_rows(dtype, what):
    """An overflowed gradient of one row changes no gradient beyond the tiles it is in."""
    o = ops()
    q, k, v, do, _ = attention_inputs((1, 500, 2, 1, 64, 20, 0, None), dtype)
    got = []
    for d in (do, do.clone()):
        if got:
            d[0, 5, 1, 7] = what
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        got.append(torch.autograd.grad(o.window_attention(*leaves, 20, 0), leaves, d))
    u = ref.half_step(dtype)
    for a, b in zip(*got):
        # rows from 256 on share no tile with row 5; fp16 may have scaled ds by another power of two
        assert torch.isfinite(b[:, 256:]).all()
        assert ref.rel(b[:, 256:], a[:, 256:].double()) <= 2 * u
    assert not torch.isfinite(got[1][0][0, 5, 1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
def test_a_large_gradient_costs_others_no_bits(dtype):
    """Gradients of 1e-3 beside one row of 3e4: dq, dk and dv of rows that share no tile with it, to the bounds of a call without it."""
    o = ops()
    q, k, v, do, _ = attention_inputs((1, 500, 2, 1, 64, 20, 0, None), dtype)
    do = do * 1e-3
    got = []
    for d in (do, do.clone()):
        if got:
            d[0, 5] = 3e4
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        got.append(torch.autograd.grad(o.window_attention(*leaves, 20, 0), leaves, d))
    for a, b in zip(*got):
        assert ref.rel(b[:, 256:], a[:, 256:].double()) <= 2 * ref.half_step(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("window, sinks, row", [(20, 4, 400), (20, 0, 200), (20, 0, 130), (20, 0, 128), (128, 130, 300), (129, 1, 300), (200, 0, 383),
                                                (200, 7, 699), (300, 3, 450), (1, 2, 257), (600, 0, 650)])
@pytest.mark.parametrize("D, group", [(64, 1), (128, 2), (72, 2)])
def test_a_large_gradient_costs_keys_that_it_does_not_meet_no_bits(dtype, window, sinks, row, D, group):
    """Gradients of 1e-3 beside one row of 3e4: dk and dv of every key that the row does not see, and dq of every other row, to
    the bounds of a call without it.  float16 results are held to 2^-24 absolute: 2^-25 / rms more, as below."""
    o = ops()
    T = 700
    q, k, v, do, _ = attention_inputs((1, T, group, 1, D, window, sinks, None), dtype)
    do = do * 1e-3
    do[0, row, 0] = 3e4
    leaves = [x.requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(o.window_attention(*leaves, window, sinks), leaves, do)
    r = [x.detach().double().requires_grad_() for x in leaves]
    dwant = torch.autograd.grad(ref.attention(*r, window, sinks), r, do.double())
    meets = ref.seen_mask(T, T, window, sinks)[row]
    rest = torch.arange(T) != row
    for name, at, got, want in zip("qkv", (rest, ~meets, ~meets), grads, dwant):
        got, want = got[0, at.cuda()].double(), want[0, at.cuda()]
        floor = 2.0 ** -25 / float(want.square().mean().sqrt()) if dtype == torch.float16 and want.any() else 0.0
        assert ref.rel(got, want) <= 5 * ref.half_step(dtype) + 256 * E + floor, "d" + name


def fp16_floor(dtype, want):
    """float16 results are held to 2^-24 absolute where they are small: 2^-25 on values of this root mean square."""
    return 2.0 ** -25 / float(want.square().mean().sqrt()) if dtype == torch.float16 and bool(want.any()) else 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("T, D, group", [(60, 128, 1), (300, 128, 1), (300, 64, 2), (700, 72, 1)])
@pytest.mark.parametrize("by", [1e-3, 1.0, 2000.0, 60000.0])
def test_gradients_over_values_of_any_size(dtype, T, D, group, by):
    """Rows of v of one sign along a gradient of ones, so that do.v is D |v| (2^23 here, and ds half of it) while the gradients
    themselves are in range: two keys a row and a small scale."""
    o = ops()
    q, k, v, do, _ = attention_inputs((1, T, group, 1, D, 2, 0, None), dtype)
    v = (torch.where(v[..., :1] < 0, -by, by) * torch.ones_like(v)).to(dtype)
    do = torch.ones_like(do)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(o.window_attention(*leaves, 2, scale=2e-4), leaves, do)
    r = [x.double().requires_grad_() for x in (q, k, v)]
    dwant = torch.autograd.grad(ref.attention(*r, 2, 0, scale=2e-4), r, do.double())
    for name, got, want in zip("qkv", grads, dwant):
        assert ref.rel(got, want) <= 5 * ref.half_step(dtype) + 256 * E + fp16_floor(dtype, want), "d" + name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("window, sinks, key", [(20, 0, 150), (20, 4, 2), (20, 4, 127), (128, 0, 128), (129, 3, 300), (200, 0, 256), (300, 200, 350)])
@pytest.mark.parametrize("D", [64, 128])
def test_a_large_value_costs_rows_that_do_not_see_it_no_bits(dtype, window, sinks, key, D):
    """Values of 1e-3 beside one of 3e4: dq of the rows that do not see it, dk of the keys that none of its rows sees, all of dv."""
    o = ops()
    T = 700
    q, k, v, do, _ = attention_inputs((1, T, 2, 1, D, window, sinks, None), dtype)
    v = v * 1e-3
    v[0, key] = 3e4
    leaves = [x.requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(o.window_attention(*leaves, window, sinks), leaves, do)
    r = [x.detach().double().requires_grad_() for x in leaves]
    dwant = torch.autograd.grad(ref.attention(*r, window, sinks), r, do.double())
    on = ref.seen_mask(T, T, window, sinks)
    rows = ~on[:, key]
    keys = ~on[on[:, key]].any(0)
    for name, at, got, want in zip("qkv", (rows, keys, torch.ones(T, dtype=torch.bool)), grads, dwant):
        got, want = got[0, at.cuda()].double(), want[0, at.cuda()]
        assert ref.rel(got, want) <= 5 * ref.half_step(dtype) + 256 * E + fp16_floor(dtype, want), "d" + name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES[1:], ids=ids_of)
def test_value_gradients_of_rows_of_many_keys(dtype):
    """Equal scores: p = 1 / (i + 1), down to 2^-18.6, and dv_j = sum of do_i / (i + 1) over i >= j.  p is off by u of its own
    size whatever that is, the sums of 4e5 terms in 32 bits by far less."""
    o = ops()
    T = 400000
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(1, T, 1, 64, generator=g, device="cuda").to(dtype) for _ in range(2))
    do = (torch.randn(1, T, 1, 64, generator=g, device="cuda") * 64).to(dtype)
    q = torch.zeros_like(k)
    v.requires_grad_()
    (dv,) = torch.autograd.grad(o.window_attention(q, k, v, T), v, do)
    terms = do[0, :, 0].double() / torch.arange(1, T + 1, device="cuda").double()[:, None]
    want = terms.flip(0).cumsum(0).flip(0)
    for lo, hi in ((0, T // 4), (T // 4, T // 2), (T // 2, 3 * T // 4)):
        assert ref.rel(dv[0, lo:hi, 0], want[lo:hi]) <= 3 * ref.half_step(dtype) + 256 * E


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("what", [float("inf"), float("nan")])
def test_what_is_not_finite_is_not_hidden(dtype, what):
    """A query, or a key that rows see, that is not finite: NaN in those rows, on every path, and no others of the head's tiles."""
    o = ops()
    for T, D in ((20, 64), (300, 64), (300, 128), (150, 33)):
        q, k, v, _, _ = attention_inputs((2, T, 2, 1, D, 8, 0, None), dtype)
        q[0, 10, 1] = what
        out = o.window_attention(q, k, v, 8)
        assert torch.isnan(out[0, 10, 1]).all()
        assert torch.isfinite(out[1]).all() and torch.isfinite(out[0, :, 0]).all() and torch.isfinite(out[0, :10, 1]).all()
        assert torch.isfinite(out[0, 11:, 1]).all()
    for T, H, Hkv, D, window in ((40, 2, 2, 64, 40), (3000, 4, 1, 64, 3000), (3000, 16, 2, 128, 2500), (3000, 2, 2, 33, 3000)):
        g = gen(T + D)
        q, k, v = randn(g, 2, H, D, dtype=dtype), randn(g, 2, T, Hkv, D, dtype=dtype), randn(g, 2, T, Hkv, D, dtype=dtype)
        n = torch.tensor([T, T], dtype=torch.int32).cuda()
        q[0, 0] = what
        out = o.window_attention_decode(q, k, v, n, window)
        assert torch.isnan(out[0, 0]).all() and torch.isfinite(out[1]).all() and torch.isfinite(out[0, 1:]).all()
        q[0, 0] = 1.0
        v[0, T - 3] = what
        out = o.window_attention_decode(q, k, v, n, window)
        assert not torch.isfinite(out[0]).any() and torch.isfinite(out[1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("what", [float("inf"), float("nan")])
@pytest.mark.parametrize("T, D", [(40, 64), (200, 64), (200, 128), (300, 72)])
def test_gradients_of_rows_that_are_not_finite(dtype, what, T, D):
    """A key or a query that is not finite makes NaN of the rows that meet it, and of the values' gradients of all keys that
    those rows see (p is NaN there): of those and of no others."""
    o = ops()
    window = 8
    for bad in "kq":
        q, k, v, do, _ = attention_inputs((1, T, 1, 1, D, window, 0, None), dtype)
        {"q": q, "k": k}[bad][0, 10] = what
        leaves = [x.requires_grad_() for x in (q, k, v)]
        out = o.window_attention(*leaves, window)
        dq, dk, dv = torch.autograd.grad(out, leaves, do)
        rows = range(10, 11) if bad == "q" else range(10, 10 + window)
        assert torch.isnan(out[0, rows]).all() and int(torch.isfinite(out[0, :, 0, 0]).sum()) == T - len(rows)
        assert torch.isnan(dq[0, rows]).all()
        keys = sorted({j for i in rows for j in range(i - window + 1, i + 1)})
        assert not torch.isfinite(dv[0, keys]).any() and not torch.isfinite(dk[0, keys]).any()
        others = [j for j in range(T) if j not in keys]
        assert torch.isfinite(dv[0, others]).all()


@pytest.mark.gpu
def test_the_first_cuda_call_of_a_thread():
    """A thread in which no context is current yet: the tile loads' descriptors need one."""
    o = ops()
    q, k, v, do, _ = attention_inputs((1, 200, 2, 2, 64, 50, 0, None), torch.bfloat16)
    lengths = torch.tensor([150], dtype=torch.int32).cuda()
    cache = randn(gen(5), 1, 2000, 2, 64, dtype=torch.bfloat16)

    def forward():
        with torch.no_grad():
            return o.window_attention(q, k, v, 50, 0)

    def both():
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        return torch.autograd.grad(o.window_attention(*leaves, 50, 0), leaves, do)[0]

    for call in (forward, both, lambda: o.window_attention_decode(q[:, 0], cache, cache, lengths, 2000)):
        want, got, errors = call(), [], []

        def run():
            try:
                got.append(call())
            except Exception as e:
                errors.append(e)

        thread = threading.Thread(target=run)
        thread.start()
        thread.join()
        assert not errors and torch.equal(got[0], want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
def test_window_attention_ignores_what_lies_behind(dtype):
    """NaN and infinity behind a sequence's length reach no output."""
    o = ops()
    for D in (64, 128, 33):
        case = (2, 200, 4, 2, D, 70, 5, [131, 64])
        q, k, v, do, n = attention_inputs(case, dtype)
        clean = [x.clone().requires_grad_() for x in (q, k, v)]
        out = o.window_attention(*clean, 70, 5, lengths=n)
        want = torch.autograd.grad(out, clean, do)
        dirty = [x.clone() for x in (q, k, v, do)]
        for x in dirty:
            for b, m in enumerate(n.tolist()):
                x[b, m:] = float("nan")
                x[b, m + 3:m + 9] = float("inf")
                x[b, m + 11:] = torch.finfo(dtype).min
        leaves = [x.requires_grad_() for x in dirty[:3]]
        got_out = o.window_attention(*leaves, 70, 5, lengths=n)
        got = torch.autograd.grad(got_out, leaves, dirty[3])
        assert torch.equal(got_out, out)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
def test_window_attention_strides(dtype):
    """Parts of one projection, heads before tokens, elements apart, rows off
    16-byte addresses, broadcast keys and gradients."""
    o = ops()
    B, T, H, D = 2, 150, 4, 64
    g = gen(9)
    u = ref.half_step(dtype)
    fused = randn(g, B, T, 3 * H * D, dtype=dtype)
    q, k, v = (x.view(B, T, H, D) for x in fused.split(H * D, 2))
    off = randn(g, B * T * H * D + 1, dtype=dtype)[1:].view(B, T, H, D)
    bhtd = randn(g, B, H, T, D, dtype=dtype).transpose(1, 2)
    apart = randn(g, B, T, D, H, dtype=dtype).transpose(2, 3)
    wide = randn(g, B, T, H, D + 4, dtype=dtype)[..., :D]
    shared = randn(g, 1, T, H, D, dtype=dtype).expand(B, T, H, D)
    one_head = randn(g, B, T, 1, D, dtype=dtype).expand(B, T, H, D)
    back = randn(g, B, T, H, D, dtype=dtype)
    for x, y, z in ((q, k, v), (off, bhtd, apart), (bhtd, off, wide), (wide, shared, one_head), (one_head, apart, shared)):
        leaves = [t.detach().requires_grad_() for t in (x, y, z)]
        for do in (back, back[:, :, :1].expand(B, T, H, D), back.transpose(1, 2).contiguous().transpose(1, 2)):
            out = o.window_attention(*leaves, 40, 3)
            grads = torch.autograd.grad(out, leaves, do)
            r = [t.detach().double().requires_grad_() for t in (x, y, z)]
            want = ref.attention(*r, 40, 3)
            dwant = torch.autograd.grad(want, r, do.double())
            assert ref.rel(out, want) <= 3 * u + 64 * E
            for got, w in zip(grads, dwant):
                assert ref.rel(got, w) <= 5 * u + 256 * E


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("by", [1e-4, 30.0])
def test_window_attention_small_and_large_gradients(dtype, by):
    """Output gradients far from 1 keep their relative accuracy (in 16 bits the
    products' operands are scaled where the type's range is short).  float16
    gradients of 1e-4 are themselves held to 2^-25 / 1e-4 of their size, inputs
    here, and dq, dk and dv of that size to the same: 2^-24 absolute on values
    whose root mean square is rms adds 2^-25 / rms."""
    o = ops()
    case = (1, 300, 2, 1, 64, 120, 4, None)
    q, k, v, do, _ = attention_inputs(case, dtype)
    do = (do.float() * by).to(dtype)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(o.window_attention(*leaves, 120, 4), leaves, do)
    r = [x.detach().double().requires_grad_() for x in leaves]
    dwant = torch.autograd.grad(ref.attention(*r, 120, 4), r, do.double())
    for got, w in zip(grads, dwant):
        floor = 2.0 ** -25 / float(w.square().mean().sqrt()) if dtype == torch.float16 else 0.0
        assert ref.rel(got, w) <= 5 * ref.half_step(dtype) + 256 * E + floor


@pytest.mark.gpu
def test_window_attention_against_differences():
    """The float32 gradients against central differences of the 64-bit form
    along random directions: a step of 1e-5 leaves 1e-9 of the differences'
    own error, far below the 256 e of the gradients (relative to the norm of
    gradient times direction)."""
    o = ops()
    case = (2, 37, 4, 2, 16, 9, 2, [37, 20])
    q, k, v, do, n = attention_inputs(case, torch.float32)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(o.window_attention(*leaves, 9, 2, lengths=n), leaves, do)
    g = gen(3)
    for at in range(3):
        base = [x.detach().double() for x in leaves]
        d = randn(g, *base[at].shape).double()
        f = []
        for h in (1e-5, -1e-5):
            moved = list(base)
            moved[at] = base[at] + h * d
            f.append(float((ref.attention(*moved, 9, 2, n) * do.double()).sum()))
        slope = (f[0] - f[1]) / 2e-5
        got = float((grads[at].double() * d).sum())
        assert abs(got - slope) <= 256 * E * float(grads[at].norm() * d.norm())


@pytest.mark.gpu
def test_window_attention_extreme_scores():
    """Scores of several hundred: one key takes all, no overflow; scores of
    -inf from finite inputs' overflow do not occur in 32 bits."""
    o = ops()
    for dtype in TYPES:
        case = (1, 200, 2, 2, 64, 90, 2, None)
        q, k, v, do, _ = attention_inputs(case, dtype, by=8.0)
        v, do = v / 8, do / 8
        out = o.window_attention(q, k, v, 90, 2)
        # scores of up to |s| = 64 * 8 * 8 * 4 / 8 = 1024 carry s * 2e in the exponent
        assert ref.rel(out, ref.attention(q, k, v, 90, 2)) <= 3 * ref.half_step(dtype) + 2048 * 2 * E


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0])
def test_window_attention_scale(dtype, scale):
    o = ops()
    case = (1, 200, 2, 1, 64, 90, 2, None)
    q, k, v, do, _ = attention_inputs(case, dtype)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = o.window_attention(*leaves, 90, 2, scale=scale)
    grads = torch.autograd.grad(out, leaves, do)
    r = [x.detach().double().requires_grad_() for x in leaves]
    want = ref.attention(*r, 90, 2, scale=scale)
    dwant = torch.autograd.grad(want, r, do.double())
    u = ref.half_step(dtype)
    assert ref.rel(out, want) <= 3 * u + 64 * E
    for got, w in zip(grads, dwant):
        assert ref.rel(got, w) <= 5 * u + 256 * E
    n = torch.tensor([150], dtype=torch.int32).cuda()
    got = o.window_attention_decode(q[:, 149].detach(), k.detach(), v.detach(), n, 90, 2, scale=scale)
    assert ref.rel(got, ref.decode(q[:, 149].detach(), k.detach(), v.detach(), n, 90, 2, scale)) <= 3 * u + 64 * E


@pytest.mark.gpu
def test_a_wait_that_ran_out_is_reported_by_the_next_call():
    """The word that a kernel sets when a wait of its runs out is set here from
    the host: the next call fails once, with its text, and the one after runs."""
    import ctypes
    import os

    from conftest import LIB

    o = ops()
    q = torch.randn(1, 200, 2, 64, device="cuda").bfloat16()
    want = o.window_attention(q, q, q, 50)
    lib = ctypes.CDLL(os.path.join(LIB, "libcail_ops.so"))
    lib.cail_ops_device_error_word.restype = ctypes.POINTER(ctypes.c_int)
    word = lib.cail_ops_device_error_word(torch.cuda.current_device())
    assert word and word[0] == 0
    word[0] = 1
    with pytest.raises(RuntimeError, match="gave up waiting"):
        o.window_attention(q, q, q, 50)
    assert word[0] == 0 and torch.equal(o.window_attention(q, q, q, 50), want)
    assert not lib.cail_ops_device_error_word(-1)


@pytest.mark.gpu
def test_window_attention_empty():
    o = ops()
    for shape in ((0, 4, 2, 8), (2, 0, 2, 8)):
        x = torch.zeros(*shape).cuda().requires_grad_()
        out = o.window_attention(x, x, x, 3)
        assert out.shape == shape
        assert torch.autograd.grad(out, x, torch.zeros_like(out))[0].shape == shape
    x = torch.zeros(2, 5, 2, 8).cuda().requires_grad_()
    out = o.window_attention(x, x, x, 3, lengths=torch.tensor([-4, 99], dtype=torch.int32).cuda())
    assert not out.any()
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(out.sum(), x, create_graph=True)


DECODE = [
    # B, T, H, Hkv, D, window, sinks, lengths
    (1, 1, 1, 1, 16, 1, 0, [1]),
    (3, 9, 2, 2, 64, 4, 2, [9, 0, 1]),
    (2, 300, 6, 2, 64, 100, 5, [300, 99]),
    (2, 300, 4, 1, 128, 1000, 0, [300, 257]),
    (1, 2000, 16, 2, 128, 1500, 130, [1999]),
    (4, 70, 5, 1, 33, 16, 3, [70, 17, 16, 2]),
    (2, 130, 9, 1, 80, 64, 300, [130, 128]),
    (1, 5000, 1, 1, 64, 5000, 0, [5000]),
    (2, 40, 3, 3, 8, 7, 1, [-3, 99]),
    (3, 1300, 5, 1, 64, 1111, 17, [1300, 1128, 900]),
    (1, 3000, 20, 1, 128, 2500, 33, [2999]),
    (2, 2048, 1, 1, 72, 2048, 0, [2048, 0]),
    (2, 1500, 4, 1, 128, 300, 300, [1500, 512]),
    (1, 9000, 2, 2, 40, 9000, 5, [8999]),
    (5, 1100, 2, 2, 64, 1024, 16, [1100, 1024, 1040, 1, 0]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("case", DECODE, ids=str)
def test_decode_matches_64_bit(dtype, case):
    o = ops()
    B, T, H, Hkv, D, window, sinks, lengths = case
    g = gen(T)
    q, k, v = randn(g, B, H, D, dtype=dtype), randn(g, B, T, Hkv, D, dtype=dtype), randn(g, B, T, Hkv, D, dtype=dtype)
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    want = ref.decode(q, k, v, n, window, sinks)
    u = ref.half_step(dtype)
    got = o.window_attention_decode(q, k, v, n, window, sinks)
    assert ref.rel(got, want) <= 3 * u + 64 * E
    # what it does not see may hold anything: other rows, and caches in other layouts
    for c in (k, v):
        for b, m in enumerate(lengths):
            m = min(max(m, 0), T)
            c[b, m:] = float("nan")
            c[b, sinks:max(sinks, m - window)] = float("inf")
    assert torch.equal(o.window_attention_decode(q, k, v, n, window, sinks), got)
    kt, vt = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    assert torch.equal(o.window_attention_decode(q, kt, vt, n, window, sinks), got)
    off = torch.empty(k.numel() + 1, dtype=dtype, device="cuda")[1:].view(k.shape).copy_(k)
    assert ref.rel(o.window_attention_decode(q, off, v, n, window, sinks), want) <= 3 * u + 64 * E


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES[1:], ids=ids_of)
@pytest.mark.parametrize("H, Hkv, D", [(2, 2, 64), (32, 8, 128), (8, 1, 64), (7, 1, 128), (9, 1, 64), (16, 1, 128), (20, 1, 80), (32, 2, 64)])
@pytest.mark.parametrize("T, window, sinks", [(4000, 3000, 4), (1300, 1300, 0), (300, 40, 20)])
def test_decode_loses_one_rounding(dtype, H, Hkv, D, T, window, sinks):
    """Element by element: o is off by its own rounding; p reaches its sum to 2 u^2 and 256 E (exponentials and sums of up to 3000
    terms in 32 bits) relative to the terms p |v|, and float16 holds small results to 2^-25."""
    o = ops()
    g = gen(T + H)
    q, k, v = randn(g, 2, H, D, dtype=dtype, by=2.0), randn(g, 2, T, Hkv, D, dtype=dtype), randn(g, 2, T, Hkv, D, dtype=dtype)
    n = torch.tensor([T, T - 77], dtype=torch.int32).cuda()
    got = o.window_attention_decode(q, k, v, n, window, sinks).double()
    want, size = ref.decode(q, k, v, n, window, sinks), ref.decode(q, k, v.abs(), n, window, sinks)
    u = ref.half_step(dtype)
    small = 2.0 ** -25 if dtype == torch.float16 else 0.0
    assert ((got - want).abs() <= u * want.abs() * (1 + u) + (2 * u * u + 256 * E) * size * (1 + u) + small).all()


@pytest.mark.gpu
def test_decode_past_32_bit_offsets():
    """A cache of more than 2^32 bytes and 2^31 elements: the last token of the
    last sequence."""
    o = ops()
    B, T, H, D = 3, 1 << 20, 8, 128
    k = torch.zeros(B, T, H, D, dtype=torch.bfloat16, device="cuda")
    assert k.numel() > 2 ** 31
    g = gen(2)
    tail = randn(g, 40, H, D, dtype=torch.bfloat16)
    k[2, -40:] = tail
    q = randn(g, B, H, D, dtype=torch.bfloat16)
    n = torch.tensor([0, 3, T], dtype=torch.int32).cuda()
    got = o.window_attention_decode(q, k, k, n, 40)
    want = ref.decode(q[2:], tail[None], tail[None], [40], 40, 0)
    assert ref.rel(got[2:], want) <= 3 * ref.half_step(torch.bfloat16) + 64 * E
    assert not got[:2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
def test_decode_is_the_last_row_of_attention(dtype):
    o = ops()
    case = (3, 190, 4, 2, 64, 50, 6, [190, 51, 7])
    q, k, v, _, n = attention_inputs(case, dtype)
    full = o.window_attention(q, k, v, 50, 6, lengths=n)
    last = torch.stack([q[b, m - 1] for b, m in enumerate(case[7])])
    got = o.window_attention_decode(last, k, v, n, 50, 6)
    for b, m in enumerate(case[7]):
        assert ref.rel(got[b], full[b, m - 1]) <= 4 * ref.half_step(dtype) + 128 * E


# -------------------------------------------------------------- distillation

# N, V, K, tau, hard, targets, gone entries
DISTILL = [
    (1, 1, 1, 1.0, 0.0, False, 0.0),
    (2, 7, 3, 2.0, 0.5, True, 0.0),
    (5, 257, 257, 1.0, 1.0, True, 0.3),
    (3, 513, 1, 3.7, 0.25, True, 0.0),
    (7, 1001, 20, 2.0, 0.0, True, 0.5),
    (4, 50257, 33, 1.0, 0.5, True, 0.1),
    (2, 50257, 64, 2.0, 0.3, True, 0.0),
    (3, 32768, 1024, 0.7, 0.9, True, 0.2),
    (2, 65537, 16, 1.5, 0.0, False, 1.0),
    (6, 100, 0, 1.0, 0.5, True, 0.0),
]

# enough rows for the kernels that stream them: rows of one and several pieces, odd lengths, more rows than blocks, K at its largest
DISTILL_MANY = [
    (150, 8193, 5, 2.0, 0.5, True, 0.2),
    (700, 8200, 33, 1.0, 0.3, True, 0.0),
    (460, 20011, 129, 3.0, 0.5, True, 0.3),
    (160, 17001, 1024, 2.0, 0.7, True, 0.1),
    (300, 9001, 16, 1.7, 0.0, False, 0.5),
    (200, 16387, 12, 1.0, 1.0, True, 0.0),
]


def distill_inputs(case, dtype, seed=0):
    N, V, K, tau, hard, has_y, gone = case
    g = gen(seed + V)
    z = randn(g, N, V, dtype=dtype, by=2.0)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(N)])
    ids[torch.rand(N, K, generator=g) < gone] = -1
    t = randn(g, N, K, by=1.5)
    y = torch.randint(0, V, (N,), generator=g).cuda() if has_y else None
    if has_y and N > 2:
        y[1], y[2] = -100, V
    if K > 3:
        ids[0, 2] = ids[0, 0]  # the same id twice
        if has_y:
            ids[0, 3] = y[0]
        ids[-1, 1] = V + 5
    return z, ids.cuda(), t, y


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("case", DISTILL, ids=str)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_distill_matches_64_bit(dtype, case, reduction):
    o = ops()
    N, V, K, tau, hard = case[:5]
    z, ids, t, y = distill_inputs(case, dtype)
    kw = dict(temperature=tau, hard_weight=hard, reduction=reduction)
    with torch.no_grad():
        plain = o.distill_loss(z, ids, t, y, **kw)
    z.requires_grad_()
    loss = o.distill_loss(z, ids, t, y, **kw)
    assert torch.equal(loss, plain) and loss.dtype == torch.float32
    g = randn(gen(1), *loss.shape) if reduction == "none" else torch.tensor(256.0).cuda()
    (dz,) = torch.autograd.grad(loss, z, g)
    r = z.detach().double().requires_grad_()
    want = ref.distill(r, ids, t, y, tau, hard, reduction)
    assert float((loss.double() - want).abs().max()) <= 2e-6 * (1 + float(want.abs().max())) * (N if reduction == "sum" else 1)
    if want.requires_grad:
        (dwant,) = torch.autograd.grad(want, r, g.double())
    else:
        dwant = torch.zeros_like(r)
    # float16: values below its smallest normal carry 2^-25 each, absolute
    floor = 2.0 ** -25 * dz.numel() ** 0.5 / max(float(dwant.norm()), 1e-30) if dtype == torch.float16 else 0.0
    assert dz.dtype == dtype and ref.rel(dz, dwant) <= ref.half_step(dtype) + 64 * E + floor
    if y is not None and N > 2:
        assert not dz[1:3].any()
    (again,) = torch.autograd.grad(o.distill_loss(z, ids, t, y, **kw), z, g)
    assert torch.equal(again, dz)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("case", DISTILL_MANY, ids=str)
def test_distill_many_rows(dtype, case):
    """Loss, gradient and both again on rows further apart; the form of many
    rows at once, built on torch's log_softmax in 64 bits."""
    o = ops()
    N, V, K, tau, hard, has_y, gone = case
    g = torch.Generator(device="cuda").manual_seed(V)
    z = (torch.randn(N, V, generator=g, device="cuda") * 2).to(dtype)
    ids = torch.randint(0, V, (N, K), generator=g, device="cuda")
    ids[torch.rand(N, K, generator=g, device="cuda") < gone] = -1
    ids[::3, 0] = V - 1  # the last element, and
    ids[1::3, 0] = 0     # the first, outside the vectors of most rows
    if K > 3:
        ids[::2, 1] = ids[::2, 3]
    t = torch.randn(N, K, generator=g, device="cuda") * 1.5
    y = torch.randint(0, V, (N,), generator=g, device="cuda") if has_y else None
    if has_y:
        y[::7] = -100
        y[1::7] = 0
        y[2::7] = V - 1
        if K > 3:
            ids[3::7, 2] = y[3::7]
    r = z.double().requires_grad_()
    counts = torch.ones(N, dtype=torch.bool, device="cuda") if y is None else (y >= 0) & (y < V)
    ok = (ids >= 0) & (ids < V)
    p = torch.where(ok, torch.softmax(torch.where(ok, t.double() / tau, -1e300), 1), 0.0)
    lq = torch.log_softmax(r / tau, 1).gather(1, ids.clamp(min=0))
    rows = (1 - hard) * tau * tau * (torch.special.xlogy(p, p) - p * lq).sum(1)
    if hard:
        rows = rows - hard * torch.log_softmax(r, 1).gather(1, y.clamp(min=0)[:, None])[:, 0]
    want = torch.where(counts, rows, 0.0).sum() / counts.sum()
    (dwant,) = torch.autograd.grad(want, r, torch.tensor(512.0, dtype=torch.float64).cuda())
    tol = ref.half_step(dtype) + 64 * E
    floor = 2.0 ** -25 * dwant.numel() ** 0.5 / float(dwant.norm()) if dtype == torch.float16 else 0.0
    wide = torch.zeros(N, V + 24, dtype=dtype, device="cuda")
    wide[:, 5:V + 5] = z
    for x in (z, wide[:, 5:V + 5]):
        x = x.detach().requires_grad_()
        loss = o.distill_loss(x, ids, t, y, temperature=tau, hard_weight=hard)
        (dz,) = torch.autograd.grad(loss, x, torch.tensor(512.0).cuda())
        assert abs(float(loss.detach()) - float(want.detach())) <= 2e-6 * (1 + float(want.detach()))
        assert ref.rel(dz, dwant) <= tol + floor
        assert not dz[~counts].any()
        # element by element: a misplaced term of one entry does not drown in the norm
        err = (dz.double() - dwant).abs()
        assert float((err - (tol * dwant.abs() + 64 * E * 512 / float(counts.sum()) + 2.0 ** -24)).max()) <= 0
        (again,) = torch.autograd.grad(o.distill_loss(x, ids, t, y, temperature=tau, hard_weight=hard), x, torch.tensor(512.0).cuda())
        assert torch.equal(again, dz)
    assert torch.equal(wide[:, :5], torch.zeros_like(wide[:, :5])) and not wide[:, V + 5:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("N, V", [(5, 301), (6, 30011), (200, 20003)])
@pytest.mark.parametrize("tau", [1.0, 2.0, 3.0])
def test_distill_hides_nothing_that_is_not_finite(dtype, N, V, tau):
    """NaN or plus infinity in a row of logits or among the teacher's, a row of minus infinity: no finite loss or gradient for
    that row, and the others' bits unchanged."""
    o = ops()
    g = gen(N + V)
    z, t = randn(g, N, V, dtype=dtype), randn(g, N, 5)
    ids, y = torch.randint(0, V, (N, 5), generator=g).cuda(), torch.randint(0, V, (N,), generator=g).cuda()

    def run(z, t):
        z = z.clone().requires_grad_()
        loss = o.distill_loss(z, ids, t, y, temperature=tau, hard_weight=0.5, reduction="none")
        return loss.detach(), torch.autograd.grad(loss.sum(), z)[0]

    loss, grad = run(z, t)
    assert torch.isfinite(loss).all() and torch.isfinite(grad).all()
    others = torch.arange(N).cuda() != 3
    nan, inf = float("nan"), float("inf")
    cases = [(z, (3, 0), nan), (z, (3, V - 1), nan), (z, (3, V // 2), inf), (z, 3, -inf), (t, (3, 2), nan), (t, (3, 2), inf), (t, 3, nan),
             (t, 3, -inf)]
    for of, at, what in cases:
        zz, tt = z.clone(), t.clone()
        (tt if of is t else zz)[at] = what
        l, d = run(zz, tt)
        assert not torch.isfinite(l[3])
        assert not torch.isfinite(d[3]).all()
        assert torch.equal(l[others], loss[others]) and torch.equal(d[others], grad[others])


@pytest.mark.gpu
def test_distill_strides_types_and_padding():
    """Rows of a wider projection (padded vocabulary), rows off 16 bytes,
    transposed logits, 32-bit ids and targets, 16-bit teachers, logits of -inf
    in a padded vocabulary, rows that are left out and hold NaN."""
    o = ops()
    case = (6, 333, 9, 2.0, 0.5, True, 0.2)
    for dtype in TYPES:
        z, ids, t, y = distill_inputs(case, dtype)
        tol = ref.half_step(dtype) + 64 * E
        wide = torch.full((6, 350), 7.0, dtype=dtype, device="cuda")
        wide[:, 3:336] = z
        off = torch.zeros(6 * 333 + 1, dtype=dtype, device="cuda")[1:].view(6, 333).copy_(z)
        far = torch.zeros(6, 2000, dtype=dtype, device="cuda")
        far[:, 1:334] = z
        for x in (wide[:, 3:336], z.T.contiguous().T, off, far[:, 1:334], wide[:, 3:336][:1].expand(6, 333)):
            x = x.detach().requires_grad_()
            loss = o.distill_loss(x, ids.int(), t, y.int(), temperature=2.0, hard_weight=0.5)
            (dz,) = torch.autograd.grad(loss, x)
            r = x.detach().double().requires_grad_()
            want = ref.distill(r, ids, t, y, 2.0, 0.5)
            (dwant,) = torch.autograd.grad(want, r)
            floor = 2.0 ** -25 * dz.numel() ** 0.5 / float(dwant.norm()) if dtype == torch.float16 else 0.0
            assert abs(float(loss) - float(want)) <= 2e-5 and ref.rel(dz, dwant) <= tol + floor
        for tt in (t.bfloat16(), t.half()):
            a = o.distill_loss(z, ids, tt, y, temperature=2.0, hard_weight=0.5)
            assert abs(float(a) - float(ref.distill(z, ids, tt, y, 2.0, 0.5))) <= 2e-5
        padded = torch.full((6, 400), float("-inf"), dtype=dtype, device="cuda")
        padded[:, :333] = z
        padded[1] = float("nan")  # a row that is left out
        padded.requires_grad_()
        loss = o.distill_loss(padded, ids.where(ids < 333, -1), t, y.where(y < 333, -1), temperature=2.0, hard_weight=0.5)
        (dz,) = torch.autograd.grad(loss, padded)
        x = z.clone().requires_grad_()
        same = o.distill_loss(x, ids, t, y, temperature=2.0, hard_weight=0.5)
        (dx,) = torch.autograd.grad(same, x)
        assert abs(float(loss) - float(same)) <= 4e-6
        assert not dz[:, 333:].any() and not dz[1].any() and ref.rel(dz[:, :333], dx) <= 2 * tol


@pytest.mark.gpu
def test_distill_against_differences():
    """The float32 gradient against central differences of the 64-bit form."""
    o = ops()
    for case in ((4, 57, 6, 2.0, 0.5, True, 0.2), (3, 40, 5, 1.3, 0.0, False, 0.0)):
        z, ids, t, y = distill_inputs(case, torch.float32)
        z.requires_grad_()
        (dz,) = torch.autograd.grad(o.distill_loss(z, ids, t, y, temperature=case[3], hard_weight=case[4]), z)
        d = randn(gen(4), *z.shape).double()
        f = [float(ref.distill(z.detach().double() + h * d, ids, t, y, case[3], case[4])) for h in (1e-5, -1e-5)]
        assert abs((f[0] - f[1]) / 2e-5 - float((dz.double() * d).sum())) <= 64 * E * float(dz.norm() * d.norm()) + 1e-8


@pytest.mark.gpu
def test_distill_empty_and_nothing_counts():
    o = ops()
    z = torch.zeros(0, 9).cuda().requires_grad_()
    e, t = torch.zeros(0, 2, dtype=torch.int64).cuda(), torch.zeros(0, 2).cuda()
    loss = o.distill_loss(z, e, t)
    assert float(loss) == 0.0 and torch.autograd.grad(loss, z)[0].shape == (0, 9)
    z = randn(gen(1), 3, 9).requires_grad_()
    loss = o.distill_loss(z, torch.zeros(3, 2, dtype=torch.int64).cuda(), torch.zeros(3, 2).cuda(), torch.full((3,), -100).cuda(), hard_weight=0.5)
    assert float(loss) == 0.0 and not torch.autograd.grad(loss, z)[0].any()
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(o.distill_loss(z, torch.zeros(3, 2, dtype=torch.int64).cuda(), torch.zeros(3, 2).cuda()), z, create_graph=True)


def distill_rows(z, ids, t, y, tau, hard):
    """The rows' losses in 64 bits, many rows at once; y within the vocabulary, a valid teacher entry in every row."""
    ok = (ids >= 0) & (ids < z.size(1))
    p = torch.where(ok, torch.softmax(torch.where(ok, t.double() / tau, -1e300), 1), 0.0)
    lq = torch.log_softmax(z / tau, 1).gather(1, ids.clamp(min=0))
    soft = (torch.special.xlogy(p, p) - torch.where(ok, p * lq, 0.0)).sum(1)
    return (1 - hard) * tau * tau * soft - hard * torch.log_softmax(z, 1).gather(1, y[:, None])[:, 0]


def check_distill_rows(z, ids, t, y, tau, hard=0.3):
    o = ops()
    z = z.detach().requires_grad_()
    loss = o.distill_loss(z, ids, t, y, temperature=tau, hard_weight=hard, reduction="none")
    (dz,) = torch.autograd.grad(loss, z, torch.full_like(loss, 64.0))
    r = z.detach().double().requires_grad_()
    want = distill_rows(r, ids, t, y, tau, hard)
    (dwant,) = torch.autograd.grad(want, r, torch.full_like(want, 64.0))
    assert float((loss.double() - want).abs().max()) <= 2e-6 * (1 + float(want.abs().max()))
    floor = 2.0 ** -25 * dz.numel() ** 0.5 / float(dwant.norm()) if z.dtype == torch.float16 else 0.0
    assert ref.rel(dz, dwant) <= ref.half_step(z.dtype) + 64 * E + floor


# V of less than a block's threads, of a row for several blocks, and rows that stream
DISTILL_RANGES = [(3, 301), (6, 30011), (200, 20003)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("N, V", DISTILL_RANGES)
@pytest.mark.parametrize("tau", [1.0, 2.0, 3.0, 0.5])
def test_distill_does_not_depend_on_what_rows_have_in_common(dtype, N, V, tau):
    """Logits and teachers' logits around -100, -1e4, 1e4: both are differences from the row's reference before anything is
    rounded (exact where they lie within a factor of two), so the bounds are those of logits around 0."""
    g = gen(N + V)
    z, t = randn(g, N, V, by=2.0), randn(g, N, 7, by=1.5)
    ids, y = torch.randint(0, V, (N, 7), generator=g).cuda(), torch.randint(0, V, (N,), generator=g).cuda()
    for shift in (-50.0, -100.0, -200.0, -1e4, 300.0, 1e4):
        check_distill_rows((z + shift).to(dtype), ids, t + shift, y, tau)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=ids_of)
@pytest.mark.parametrize("N, V", DISTILL_RANGES)
@pytest.mark.parametrize("tau", [1.0, 2.0, 3.0, 0.5])
def test_distill_over_a_masked_vocabulary(dtype, N, V, tau):
    """A third of the vocabulary at -1e4 or at the type's lowest value, at the row's start, middle or end, and a row of nothing
    else (equal logits: log V)."""
    g = gen(N + V + 1)
    z, t = randn(g, N, V, dtype=dtype, by=2.0), randn(g, N, 7, by=1.5)
    for fill in (-1e4, torch.finfo(dtype).min):
        for lo, hi in ((0, V // 3), (V // 3, 2 * V // 3), (2 * V // 3, V)):
            x = z.clone()
            x[:, lo:hi] = fill
            ids, y = (torch.randint(0, V - hi + lo, s, generator=g).cuda() for s in ((N, 7), (N,)))
            ids, y = (torch.where(i < lo, i, i + hi - lo) for i in (ids, y))  # outside the masked third
            check_distill_rows(x, ids, t, y, tau)
            if lo:
                x[1] = fill
                check_distill_rows(x, ids, t, y, tau)


# ------------------------------------------------- streams, graphs, together


def step(o, x, plan, window, sinks, n, ids, t, y):
    """rotary, attention, a projection and the loss: a model's tail in small."""
    q, k, v, w = x
    qr, kr = o.rotary(q, k, plan)
    a = o.window_attention(qr, kr, v, window, sinks, lengths=n)
    logits = a.flatten(2).flatten(0, 1) @ w
    return o.distill_loss(logits, ids, t, y, temperature=2.0, hard_weight=0.5)


def step_inputs(seed, dtype=torch.bfloat16):
    g = gen(seed)
    B, T, H, D, V, K = 2, 140, 4, 64, 301, 7
    x = [randn(g, B, T, H, D, dtype=dtype), randn(g, B, T, 2, D, dtype=dtype), randn(g, B, T, 2, D, dtype=dtype),
         randn(g, H * D, V, dtype=dtype, by=0.2)]
    n = torch.tensor([140, 77], dtype=torch.int32).cuda()
    ids = torch.randint(0, V, (B * T, K), generator=g).cuda()
    y = torch.randint(0, V, (B * T,), generator=g).cuda()
    y[140 + 77:] = -100
    return x, n, ids, randn(g, B * T, K), y


@pytest.mark.gpu
def test_operators_together_match_64_bit():
    o = ops()
    plan = o.Rotary(32)
    f, amp = freqs(32)
    x, n, ids, t, y = step_inputs(1)
    leaves = [p.requires_grad_() for p in x]
    loss = step(o, leaves, plan, 50, 4, n, ids, t, y)
    grads = torch.autograd.grad(loss, leaves)
    r = [p.detach().double().requires_grad_() for p in x]
    at = torch.arange(140).cuda().expand(2, 140)
    a = ref.attention(ref.rotate(r[0], at, f, amp, False), ref.rotate(r[1], at, f, amp, False), r[2], 50, 4, n)
    want = ref.distill(a.flatten(2).flatten(0, 1) @ r[3], ids, t, y, 2.0, 0.5)
    dwant = torch.autograd.grad(want, r)
    u = ref.half_step(torch.bfloat16)
    # the loss sees logits of the order of 3 that carry a few roundings each, averaged over 217 rows
    assert abs(float(loss) - float(want)) <= 4 * u * 3
    for got, w in zip(grads, dwant):  # eight roundings to 16 bits lie between the inputs and their gradients
        assert ref.rel(got, w) <= 8 * u


@pytest.mark.gpu
def test_operators_on_another_stream_and_captured():
    """A whole step on a side stream, and captured into two graphs that are
    replayed in turn with new inputs, gives the bits of the eager step."""
    o = ops()
    plan = o.Rotary(32)
    want, data = [], [step_inputs(s) for s in (1, 2, 3)]
    for x, n, ids, t, y in data:
        leaves = [p.clone().requires_grad_() for p in x]
        loss = step(o, leaves, plan, 50, 4, n, ids, t, y)
        grads = torch.autograd.grad(loss, leaves)
        want.append((loss.detach().clone(), *grads))
        del loss, leaves
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        x, n, ids, t, y = data[1]
        leaves = [p.clone().requires_grad_() for p in x]
        loss = step(o, leaves, plan, 50, 4, n, ids, t, y)
        got = (loss.detach(), *torch.autograd.grad(loss, leaves))
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    del loss, leaves

    runs = []
    for first in (0, 1):
        x, n, ids, t, y = data[first]
        static = [p.clone().requires_grad_() for p in x] + [n.clone(), ids.clone(), t.clone(), y.clone()]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss = step(o, static[:4], plan, 50, 4, *static[4:])
            out = (loss.detach(), *torch.autograd.grad(loss, static[:4]))
            del loss
        runs.append((graph, static, out))
    for order in (0, 2, 1):
        for graph, static, out in runs:
            x, *rest = data[order]
            with torch.no_grad():
                for dst, src in zip(static, [*x, *rest]):
                    dst.copy_(src)
        for graph, _, _ in runs:
            graph.replay()
        torch.cuda.synchronize()
        for _, _, out in runs:
            assert all(torch.equal(a, b) for a, b in zip(out, want[order]))


@pytest.mark.gpu
def test_decode_captured_follows_the_lengths():
    o = ops()
    g = gen(8)
    q, k, v = randn(g, 2, 4, 64, dtype=torch.bfloat16), *(randn(g, 2, 500, 2, 64, dtype=torch.bfloat16) for _ in range(2))
    n = torch.tensor([1, 0], dtype=torch.int32).cuda()
    o.window_attention_decode(q, k, v, n, 100, 4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = o.window_attention_decode(q, k, v, n, 100, 4)
    for lengths in ([500, 37], [3, 0], [101, 104]):
        n.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, o.window_attention_decode(q, k, v, n, 100, 4))
        assert ref.rel(out, ref.decode(q, k, v, lengths, 100, 4)) <= 3 * ref.half_step(torch.bfloat16) + 64 * E


def part_of_the_sms(count):
    """A stream whose kernels run on `count` SMs (a green context of this process; nothing outlasts it)."""
    d = pytest.importorskip("cuda.bindings.driver")

    def get(r):
        if r[0] != d.CUresult.CUDA_SUCCESS:
            pytest.skip(f"no part of the SMs to be had: {r[0]}")
        return r[1] if len(r) == 2 else r[1:]

    dev = get(d.cuDeviceGet(torch.cuda.current_device()))
    sms = get(d.cuDeviceGetDevResource(dev, d.CUdevResourceType.CU_DEV_RESOURCE_TYPE_SM))
    flags = int(d.CUdevSmResourceSplit_flags.CU_DEV_SM_RESOURCE_SPLIT_IGNORE_SM_COSCHEDULING) if count < 8 else 0
    groups = get(d.cuDevSmResourceSplitByCount(1, sms, flags, count))[0]
    ctx = get(d.cuGreenCtxCreate(get(d.cuDevResourceGenerateDesc([groups[0]], 1)), dev, d.CUgreenCtxCreate_flags.CU_GREEN_CTX_DEFAULT_STREAM))
    return torch.cuda.ExternalStream(int(get(d.cuGreenCtxStreamCreate(ctx, d.CUstream_flags.CU_STREAM_NON_BLOCKING, 0))))


@pytest.mark.gpu
@pytest.mark.parametrize("sms", [2, 8, 16])
def test_clusters_on_a_part_of_the_sms(sms):
    """Where a cluster of the size that the whole GPU would have does not fit, smaller ones run: the same results but for the
    sums' order, by the bounds against 64 bits."""
    o = ops()
    g = gen(sms)
    q, k, v = randn(g, 1, 2, 64), randn(g, 1, 16384, 2, 64), randn(g, 1, 16384, 2, 64)
    n = torch.tensor([16000], dtype=torch.int32).cuda()
    z, ids, t, y = distill_inputs((2, 50257, 33, 2.0, 0.3, True, 0.1), torch.float32)
    o.window_attention_decode(q, k, v, n, 16384)
    torch.cuda.synchronize()
    with torch.cuda.stream(part_of_the_sms(sms)):
        for dtype in TYPES:
            x = [c.to(dtype) for c in (q, k, v)]
            got = o.window_attention_decode(*x, n, 16384)
            assert ref.rel(got, ref.decode(*x, n, 16384, 0)) <= 3 * ref.half_step(dtype) + 64 * E
        loss = o.distill_loss(z, ids, t, y, temperature=2.0, hard_weight=0.3)
        want = float(ref.distill(z, ids, t, y, 2.0, 0.3))
        assert abs(float(loss) - want) <= 2e-6 * (1 + want)
        torch.cuda.current_stream().synchronize()


@pytest.mark.gpu
def test_operators_from_two_threads():
    """Two threads on streams of their own, the same bits as one after the other."""
    import threading

    o = ops()
    plan = o.Rotary(32)
    data = [step_inputs(s) for s in (4, 5)]

    def run(d):
        x, n, ids, t, y = d
        leaves = [p.clone().requires_grad_() for p in x]
        loss = step(o, leaves, plan, 50, 4, n, ids, t, y)
        return (loss.detach(), *torch.autograd.grad(loss, leaves))

    want = [run(d) for d in data]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i] = run(data[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(6))
def test_window_attention_drawn(seed):
    """Sizes drawn over the range."""
    o = ops()
    r = random.Random(seed)
    for _ in range(4):
        dtype = r.choice(TYPES)
        Hkv = r.randint(1, 3)
        T = r.choice([1, r.randint(2, 60), r.randint(61, 600)])
        case = (r.randint(1, 3), T, Hkv * r.randint(1, 4), Hkv, r.choice([4, 24, 40, 64, 100, 104, 128]), r.randint(1, T + 20),
                r.choice([0, r.randint(0, T)]), None)
        q, k, v, do, _ = attention_inputs(case, dtype, seed)
        n = torch.tensor([r.randint(0, T) for _ in range(case[0])], dtype=torch.int32).cuda() if r.random() < 0.5 else None
        leaves = [x.requires_grad_() for x in (q, k, v)]
        out = o.window_attention(*leaves, *case[5:7], lengths=n)
        grads = torch.autograd.grad(out, leaves, do)
        rr = [x.detach().double().requires_grad_() for x in leaves]
        want = ref.attention(*rr, *case[5:7], n)
        dwant = torch.autograd.grad(want, rr, do.double())
        u = ref.half_step(dtype)
        assert ref.rel(out, want) <= 3 * u + 64 * E, case
        for got, w in zip(grads, dwant):
            assert ref.rel(got, w) <= 5 * u + 256 * E, case
