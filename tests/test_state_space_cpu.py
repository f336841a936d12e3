"""State-space operators on the CPU: the oracle against the formulas written out, its gradients against differences, cut
sequences against whole ones, and what the entry points of the kernels refuse before anything is launched."""
import os
import random
import shutil
import subprocess

import pytest
import torch

import ssm_ref
from distributed_rl_amd import native
from distributed_rl_amd.ops import hip, oracle


def rnd(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, dtype=torch.float64) * scale


def scan_inputs(T, B, D, N, seed=0, grads=True):
    g = torch.Generator().manual_seed(seed)
    v = dict(u=rnd(g, T, B, D), dt=rnd(g, T, B, D, scale=0.5) - 2, A=-torch.rand(D, N, generator=g, dtype=torch.float64) * 3 - 0.1,
             Bm=rnd(g, T, B, N), Cm=rnd(g, T, B, N), D=rnd(g, D), z=rnd(g, T, B, D), dt_bias=rnd(g, D, scale=0.2), h0=rnd(g, B, D, N),
             reset=(torch.rand(T, B, generator=g) < 0.2).to(torch.uint8),
             lengths=torch.randint(0, T + 1, (B,), generator=g).to(torch.int32))
    if grads:
        v.update(dy=rnd(g, T, B, D), dhT=rnd(g, B, D, N))
    return v


SCAN_KEYS = ("u", "dt", "A", "Bm", "Cm", "D", "z", "dt_bias", "h0")


@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("T,B,D,N", [(1, 1, 1, 1), (7, 4, 3, 5), (19, 3, 2, 4)])
def test_scan_oracle_and_its_gradients_are_the_formulas(T, B, D, N, softplus):
    v = scan_inputs(T, B, D, N)
    p = {k: v[k].clone().requires_grad_() for k in SCAN_KEYS}
    y, hT = oracle.ssm_scan(**p, reset=v["reset"], lengths=v["lengths"], softplus=softplus)
    ((y * v["dy"]).sum() + (hT * v["dhT"]).sum()).backward()
    ref = ssm_ref.scan(v, softplus=softplus)
    torch.testing.assert_close(y, ref["y"], rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(hT, ref["hT"], rtol=1e-12, atol=1e-12)
    for k, r in dict(u="du", dt="ddt", A="dA", Bm="dB", Cm="dC", D="dD", z="dz", dt_bias="ddt_bias", h0="dh0").items():
        torch.testing.assert_close(p[k].grad, ref[r], rtol=1e-11, atol=1e-11, msg=lambda s, k=k: "%s: %s" % (k, s))


def test_scan_gradients_against_differences():
    v = scan_inputs(6, 3, 2, 3, seed=5)
    p = [v[k].clone().requires_grad_() for k in SCAN_KEYS]
    assert torch.autograd.gradcheck(lambda *a: oracle.ssm_scan(**dict(zip(SCAN_KEYS, a)), reset=v["reset"], lengths=v["lengths"]), p)


@pytest.mark.parametrize("T,shift", [(40, -2.0), (700, -4.0)])
def test_scan_bounds_hold_for_fp32_and_not_for_a_state_of_fewer_bits(T, shift):
    v = scan_inputs(T, 3, 17, 5, seed=1)
    v["dt"] = v["dt"] * 0.6 + 2 + shift
    v = {k: x.float().double() if x.dtype == torch.float64 else x for k, x in v.items()}
    v.update(reset=(v["reset"] * (torch.arange(T) % 7 == 0)[:, None]).to(torch.uint8), lengths=torch.tensor([T, T - 9, 1], dtype=torch.int32))
    ref, tol = ssm_ref.scan(v), ssm_ref.scan_bounds(v)
    p = {k: v[k].float().requires_grad_() for k in SCAN_KEYS}
    y, hT = oracle.ssm_scan(**p, reset=v["reset"], lengths=v["lengths"])
    ((y * v["dy"].float()).sum() + (hT * v["dhT"].float()).sum()).backward()
    got = dict(y=y, hT=hT, **{r: p[k].grad for k, r in dict(u="du", dt="ddt", A="dA", Bm="dB", Cm="dC", D="dD", z="dz", dt_bias="ddt_bias", h0="dh0").items()})
    for k in got:
        ssm_ref.within(got[k], ref[k], tol[k], k)
    h, ys = v["h0"].float(), []
    for t in range(T):                                      # the oracle with its state rounded to bf16 after every step
        one = {k: v[k][t:t + 1].float() for k in ("u", "dt", "Bm", "Cm", "z")}
        y, h = oracle.ssm_scan(**one, **{k: v[k].float() for k in ("A", "D", "dt_bias")}, h0=h, reset=v["reset"][t:t + 1], lengths=v["lengths"] - t)
        h = h.bfloat16().float()
        ys.append(y[0])
    for k, x in (("y", torch.stack(ys)), ("hT", h)):
        with pytest.raises(AssertionError, match="outside"):
            ssm_ref.within(x, ref[k], tol[k], k)


def test_scan_in_pieces_is_the_whole_scan():
    v = scan_inputs(17, 3, 4, 5, seed=2, grads=False)
    v["lengths"] = None
    y, hT = oracle.ssm_scan(**v)
    cut = lambda a, b: {k: (x[a:b] if k in ("u", "dt", "Bm", "Cm", "z", "reset") else x) for k, x in v.items()}     # noqa: E731
    y1, h = oracle.ssm_scan(**cut(0, 5))
    y2, h = oracle.ssm_scan(**{**cut(5, 17), "h0": h})
    torch.testing.assert_close(torch.cat([y1, y2]), y, rtol=1e-13, atol=1e-13)
    torch.testing.assert_close(h, hT, rtol=1e-13, atol=1e-13)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_scan_oracle_over_the_whole_range_of_step_sizes(dtype):
    low = torch.finfo(dtype).min
    dt = torch.tensor([0.0, -1.0, 30.0, 45.0, 88.0, 100.0, 710.0, 800.0, 1e30, -800.0, low, float("-inf")], dtype=dtype).view(1, -1, 1)
    n = dt.shape[1]
    one = torch.ones(1, n, 1, dtype=dtype)
    x = dt.clone().requires_grad_()
    y, h = oracle.ssm_scan(one, x, -torch.ones(1, 1, dtype=dtype), one, one, h0=torch.full((n, 1, 1), 3.0, dtype=dtype))
    s = torch.logaddexp(dt.double(), torch.zeros((), dtype=torch.float64))[0]
    want = 3.0 * torch.exp(-s) + s
    # exp, log1p, their sum, the decay (its exponent's error fades with it), two products and a sum: 8 steps; twice that for the slope
    torch.testing.assert_close(y[0].double(), want, rtol=8 * torch.finfo(dtype).eps, atol=0)
    assert torch.equal(h[-2:, 0, 0], torch.full((2,), 3.0, dtype=dtype))                    # steps that are held
    y.sum().backward()
    torch.testing.assert_close(x.grad[0].double(), (1 - 3.0 * torch.exp(-s)) * torch.sigmoid(dt[0].double()), rtol=16 * torch.finfo(dtype).eps, atol=0)


def conv_inputs(T, B, D, W, seed=0):
    g = torch.Generator().manual_seed(seed)
    return dict(x=rnd(g, T, B, D), w=rnd(g, D, W), bias=rnd(g, D), state_in=rnd(g, B, W - 1, D), dy=rnd(g, T, B, D),
                dstate_out=rnd(g, B, W - 1, D), reset=(torch.rand(T, B, generator=g) < 0.25).to(torch.uint8),
                lengths=torch.randint(0, T + 1, (B,), generator=g).to(torch.int32))


@pytest.mark.parametrize("silu", [True, False])
@pytest.mark.parametrize("T,B,D,W", [(1, 2, 3, 4), (2, 5, 1, 3), (23, 4, 3, 2), (40, 6, 2, 4)])
def test_conv_oracle_and_its_gradients_are_the_formulas(T, B, D, W, silu):
    v = conv_inputs(T, B, D, W)
    p = {k: v[k].clone().requires_grad_() for k in ("x", "w", "bias", "state_in")}
    y, st = oracle.short_conv(p["x"], p["w"], p["bias"], p["state_in"], v["reset"], v["lengths"], silu)
    ((y * v["dy"]).sum() + (st * v["dstate_out"]).sum()).backward()
    ref = ssm_ref.conv(v, silu)
    for got, k in ((y, "y"), (st, "state_out"), (p["x"].grad, "dx"), (p["w"].grad, "dw"), (p["bias"].grad, "db"), (p["state_in"].grad, "dstate_in")):
        torch.testing.assert_close(got, ref[k], rtol=1e-12, atol=1e-12, msg=lambda s, k=k: "%s: %s" % (k, s))


def test_conv_gradients_against_differences():
    v = conv_inputs(6, 3, 2, 3, seed=3)
    p = [v[k].clone().requires_grad_() for k in ("x", "w", "bias", "state_in")]
    assert torch.autograd.gradcheck(lambda x, w, b, s: oracle.short_conv(x, w, b, s, v["reset"], v["lengths"]), p)


def test_norm_oracle_and_its_gradients_are_the_formulas():
    g = torch.Generator().manual_seed(0)
    v = dict(x=rnd(g, 5, 7) * 2 + 3, w=rnd(g, 7), b=rnd(g, 7), dy=rnd(g, 5, 7))
    p = [v[k].clone().requires_grad_() for k in ("x", "w", "b")]
    y = oracle.layer_norm(*p)
    (y * v["dy"]).sum().backward()
    ref = ssm_ref.norm(v)
    for got, k in ((y, "y"), (p[0].grad, "dx"), (p[1].grad, "dw"), (p[2].grad, "db")):
        torch.testing.assert_close(got, ref[k], rtol=1e-12, atol=1e-12)
    assert torch.autograd.gradcheck(lambda x, w, b: oracle.layer_norm(x, w, b), p)


# ---- refusals: raised on the host, before the library is touched ---------------------------------------------------------
def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 8), torch.ones(8)
    with pytest.raises(TypeError):
        hip.layer_norm_fwd(x, w, w, torch.empty_like(x))
    with pytest.raises(TypeError):
        hip.short_conv_fwd(x[None], torch.zeros(8, 4), w, torch.empty(1, 4, 8))
    with pytest.raises(TypeError):
        hip.short_conv_step(x, torch.zeros(8, 4), w, torch.zeros(4, 3, 8), torch.empty_like(x))
    h = torch.zeros(4, 8, 2)
    with pytest.raises(TypeError):
        hip.ssm_step(x, x.clone(), torch.zeros(8, 2), torch.zeros(4, 2), torch.zeros(4, 2), h, torch.empty_like(x))
    with pytest.raises(TypeError):
        hip.ssm_scan_fwd(x[None], x[None], torch.zeros(8, 2), torch.zeros(1, 4, 2), torch.zeros(1, 4, 2), torch.empty(1, 4, 8), torch.empty(0))


@pytest.mark.parametrize("T,B,D,N", [(0, 1, 8, 4), (3, 0, 8, 4), (3, 70000, 1, 1), (3, 1, 8, 65), (3, 1, 8, 0)])
def test_sizes_are_refused(T, B, D, N):
    u, bc = torch.empty(T, B, D), torch.empty(T, B, N)
    with pytest.raises(ValueError):
        hip.ssm_scan_fwd(u, u, torch.empty(D, N), bc, bc, u.clone(), torch.empty(0))
    with pytest.raises(ValueError):
        hip.short_conv_fwd(u, torch.empty(D, 5 if N else 1), None, u.clone())
    with pytest.raises(ValueError):
        hip.layer_norm_fwd(torch.empty(T * 0, 16385), torch.empty(16385), None, torch.empty(0, 16385))


def test_each_size_of_the_convolution_and_the_norm_is_refused_for_itself():
    for T, B, W in ((0, 3, 4), (3, 0, 4), (3, 2, 1), (3, 2, 5), (3, 2, 0)):
        u = torch.empty(T, B, 8)
        with pytest.raises(ValueError, match="short_conv: unsupported sizes"):
            hip.short_conv_fwd(u, torch.empty(8, W), None, u.clone())
    with pytest.raises(ValueError, match="short_conv: unsupported sizes"):
        hip.short_conv_fwd(torch.empty(3, 2, 0), torch.empty(0, 4), None, torch.empty(3, 2, 0))
    for W in (1, 5):
        with pytest.raises(ValueError, match="short_conv_step"):
            hip.short_conv_step(torch.empty(2, 8), torch.empty(8, W), None, torch.empty(2, 3, 8), torch.empty(2, 8))
    for M, D in ((1, 16385), (0, 8), (1, 0)):
        with pytest.raises(ValueError, match="layer_norm: x must be"):
            hip.layer_norm_fwd(torch.empty(M, D), torch.empty(D), None, torch.empty(M, D))
    with pytest.raises(TypeError, match="CUDA"):            # the largest sizes of each get as far as the device
        hip.layer_norm_fwd(torch.empty(1, 16384), torch.empty(16384), None, torch.empty(1, 16384))
    for W in (2, 4):
        with pytest.raises(TypeError, match="CUDA"):
            hip.short_conv_fwd(torch.empty(1, 1, 8), torch.empty(8, W), None, torch.empty(1, 1, 8))


def test_sizes_past_the_limits_are_refused():
    big = lambda *shape: torch.empty(1).expand(shape)                       # noqa: E731
    for T, B, D in (((1 << 30) + 1, 1, 1), (2, 65536, 1), (1, 1, (1 << 22) + 1), (40000, 65535, 1)):
        u, bc = big(T, B, D), big(T, B, 4)
        with pytest.raises(ValueError, match="unsupported sizes"):
            hip.ssm_scan_fwd(u, u, big(D, 4), bc, bc, u, torch.empty(0))
        with pytest.raises(ValueError, match="unsupported sizes"):
            hip.short_conv_fwd(u, big(D, 4), None, u)


def test_missing_tensors_are_refused():
    x, w = torch.zeros(4, 8), torch.ones(8)
    with pytest.raises(ValueError, match="w is needed"):
        hip.layer_norm_fwd(x, None, w, x.clone())
    with pytest.raises(ValueError, match="A is needed"):
        hip.ssm_step(x, x, None, x[:, :2], x[:, :2], torch.zeros(4, 8, 2), x.clone())
    with pytest.raises(ValueError, match="both or neither"):
        hip.layer_norm_fwd(x, w, w, x.clone(), mean=torch.zeros(4))
    with pytest.raises(ValueError, match="eps"):
        hip.layer_norm_fwd(x, w, w, x.clone(), eps=float("nan"))
    u = torch.zeros(2, 4, 8)
    bc = torch.zeros(2, 4, 2)
    with pytest.raises(ValueError, match="z and dz"):
        hip.ssm_scan_bwd(u, u, u, torch.zeros(8, 2), bc, bc, torch.zeros(1, 4, 8, 2), u, u, torch.zeros(8, 2), bc, bc, torch.zeros(1), z=u)
    with pytest.raises(ValueError, match="without"):
        hip.ssm_scan_bwd(u, u, u, torch.zeros(8, 2), bc, bc, torch.zeros(1, 4, 8, 2), u, u, torch.zeros(8, 2), bc, bc, torch.zeros(1), dD=w)


def test_rows_of_outputs_may_not_overlap():
    t = torch.zeros(64)
    cpu = -1                                                # the ordinal that tensors on the CPU have
    assert hip._rows(t.as_strided((2, 3, 4), (32, 8, 1)), (2, 3, 4), torch.float32, cpu, "y", True)[1:] == (32, 8)
    assert hip._rows(t.as_strided((2, 3, 4), (4, 16, 1)), (2, 3, 4), torch.float32, cpu, "y", True)[1:] == (4, 16)
    assert hip._rows(t.as_strided((2, 3, 4), (0, 0, 1)), (2, 3, 4), torch.float32, cpu, "x")[1:] == (0, 0)
    for st in ((0, 4, 1), (4, 4, 1), (8, 4, 1), (12, 3, 1), (2, 8, 1)):
        with pytest.raises(ValueError, match="overlap"):
            hip._rows(t.as_strided((2, 3, 4), st), (2, 3, 4), torch.float32, cpu, "y", True)
    with pytest.raises(ValueError, match="contiguous"):
        hip._rows(t.as_strided((2, 3, 4), (24, 8, 2)), (2, 3, 4), torch.float32, cpu, "x")
    with pytest.raises(ValueError, match="shares"):
        hip._apart((8, 0, 16), (16, 24))
    with pytest.raises(ValueError, match="shares"):
        hip._apart((8, 8), ())
    hip._apart((8, 16, 0, 0), (0, 24))


# ---- refusals past the device check: _dev is told that the CPU is the current GPU, and the arguments are only packed ----------
def scan_args(T=50, B=4, D=8, N=4, backward=False, **kw):
    z = lambda *s: torch.zeros(*s)                                          # noqa: E731
    a = dict(u=z(T, B, D), dt=z(T, B, D), A=z(D, N), Bm=z(T, B, N), Cm=z(T, B, N), D=None, z=None, dt_bias=None, softplus=True, reset=None,
             lengths=None, ws=z(64))
    a.update(dict(y=z(T, B, D)) if not backward else
             dict(ckpt=z((T + 7) // 8, B, D, N), dy=z(T, B, D), du=z(T, B, D), ddt=z(T, B, D), dA=z(D, N), dB=z(T, B, N), dC=z(T, B, N)))
    a.update(kw)
    return hip._ssm_args(**a)


@pytest.mark.parametrize("backward", [False, True])
def test_scan_coefficients_of_other_sizes_than_the_sequence_are_refused(monkeypatch, backward):
    monkeypatch.setattr(hip, "_dev", lambda t: t.get_device())
    scan_args(backward=backward)
    grads = ("dB", "dC") if backward else ()
    for shape in ((3, 1, 4), (50, 1, 4), (1, 4, 4), (49, 4, 4), (51, 4, 4), (50, 3, 4), (50, 5, 4), (4, 50, 4), (50, 4, 3)):
        both = {k: torch.zeros(shape) for k in ("Bm", "Cm") + grads}
        with pytest.raises(ValueError):                     # all of them alike: they agree with each other, not with u
            scan_args(backward=backward, **both)
        for k in both:
            with pytest.raises(ValueError):
                scan_args(backward=backward, **{k: both[k]})
    batch_major = {k: torch.zeros(4, 50, 4).transpose(0, 1) for k in ("Bm", "Cm") + grads}
    scan_args(backward=backward, **batch_major)             # a transpose of the right shape is fine


# ---- outputs that overlap ------------------------------------------------------------------------------------------------------
HARNESS = """
#include <cstdio>
#include "apart.h"
int main() {
    View v[2];
    while (true) {
        for (View& x : v)
            if (std::scanf("%lld %lld %lld %lld %lld %lld", &x.at, &x.row, &x.n[0], &x.s[0], &x.n[1], &x.s[1]) != 6) return 0;
        std::printf("%d\\n", share(v[0], v[1]));
    }
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_views_share_memory_where_their_bytes_do(tmp_path):
    src = tmp_path / "share.cpp"
    src.write_text(HARNESS)
    inc = os.path.join(os.path.dirname(hip.__file__), "..", "csrc", "hip")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", inc, str(src), "-o", str(tmp_path / "share")], check=True)
    r = random.Random(0)
    views = [((0, 8, 5, 40, 3, 200), (8, 8, 5, 40, 3, 200)),                       # neighbours in the same rows
             ((0, 8, 5, 40, 3, 200), (8, 33, 5, 40, 3, 200)),                      # ... one of them a byte too wide
             ((0, 8, 3, 200, 5, 40), (8, 8, 5, 40, 3, 200)),                       # the axes the other way round
             ((0, 4, 1000000, 0, 1, 0), (4, 4, 1000000, 0, 7, 4)),                 # one row read many times
             ((0, 2, 70000, 32768, 60000, 64), (2, 2, 70000, 32768, 60000, 64)),   # past 32 bits
             ((0, 2, 70000, 32768, 60000, 64), (2 + 69999 * 32768 + 59999 * 64, 2, 1, 0, 1, 0)),
             ((0, 2, 70000, 32768, 60000, 64), (69999 * 32768 + 59999 * 64 + 1, 2, 1, 0, 1, 0)),
             ((0, 0, 1, 0, 1, 0), (0, 8, 1, 0, 1, 0))]                             # no tensor
    want = [False, True, False, False, False, False, True, False]
    for _ in range(3000):
        one = lambda: (r.randint(0, 60), r.choice([1, 2, 4, 8]), r.randint(1, 4), r.choice([0, 3, 8, 10, 16, 24, 40]), r.randint(1, 4),   # noqa: E731
                       r.choice([0, 2, 8, 12, 16, 32, 72]))
        a, b = one(), one()
        byte = [{v[0] + i * v[3] + j * v[5] + k for i in range(v[2]) for j in range(v[4]) for k in range(v[1])} for v in (a, b)]
        views.append((a, b))
        want.append(bool(byte[0] & byte[1]))
    text = "\n".join(" ".join(map(str, a + b)) for a, b in views)
    got = subprocess.run([str(tmp_path / "share")], input=text, stdout=subprocess.PIPE, text=True, check=True, timeout=60).stdout.split()
    assert [g == "1" for g in got] == want


@pytest.mark.skipif(torch.cuda.is_available(), reason="tensors on the CPU are shown to the library as a GPU's: every call here is refused by it")
def test_outputs_that_overlap_from_another_start_are_refused(monkeypatch):
    if not native.hip_available():
        pytest.skip("libdrl_hip.so is not built")
    monkeypatch.setattr(hip, "_dev", lambda t: t.get_device())
    monkeypatch.setattr(hip, "_raw_stream", lambda dev: 0)
    z = lambda *s: torch.zeros(*s)                                          # noqa: E731
    T, B, D, N, W = 10, 3, 8, 4, 4

    def each(call, outs, ins, fixed):
        names = outs + ins
        for i, o in enumerate(outs):
            for other in names[i + 1:]:
                kw = dict(fixed)
                small, large = sorted((o, other), key=lambda k: fixed[k].nbytes)
                buf = torch.zeros(fixed[large].nbytes + 4, dtype=torch.uint8)
                for k, at in ((large, 0), (small, 4)):
                    kw[k] = buf[at:at + fixed[k].nbytes].view(fixed[k].dtype).view(fixed[k].shape)
                with pytest.raises(ValueError, match="shares"):
                    call(**kw)

    each(hip.layer_norm_fwd, ["y", "mean", "rstd"], ["x", "w", "b"], dict(x=z(T, D), w=z(D), b=z(D), y=z(T, D), mean=z(T), rstd=z(T)))
    each(hip.layer_norm_bwd, ["dx", "dw", "db", "ws"], ["dy", "x", "w", "mean", "rstd"],
         dict(dy=z(T, D), x=z(T, D), w=z(D), mean=z(T), rstd=z(T), dx=z(T, D), dw=z(D), db=z(D), ws=hip.layer_norm_ws(T, D, "cpu")))
    u8, i32 = dict(dtype=torch.uint8), dict(dtype=torch.int32)
    conv = dict(x=z(T, B, D), w=z(D, W), bias=z(D), state_in=z(B, W - 1, D), reset=torch.zeros(T, B, **u8), lengths=torch.zeros(B, **i32))
    each(hip.short_conv_fwd, ["y", "state_out"], list(conv), dict(conv, y=z(T, B, D), state_out=z(B, W - 1, D)))
    each(hip.short_conv_bwd, ["dx", "dw", "db", "dstate_in", "ws"], list(conv) + ["dy", "dstate_out"],
         dict(conv, dy=z(T, B, D), dstate_out=z(B, W - 1, D), dx=z(T, B, D), dw=z(D, W), db=z(D), dstate_in=z(B, W - 1, D),
              ws=hip.short_conv_ws(T, B, D, W, "cpu")))
    each(hip.short_conv_step, ["y", "state"], ["x", "w", "bias", "reset"],
         dict(x=z(B, D), w=z(D, W), bias=z(D), state=z(B, W - 1, D), y=z(B, D), reset=torch.zeros(B, **u8)))
    scan = dict(u=z(T, B, D), dt=z(T, B, D), A=z(D, N), Bm=z(T, B, N), Cm=z(T, B, N), D=z(D), z=z(T, B, D), dt_bias=z(D),
                reset=torch.zeros(T, B, **u8), lengths=torch.zeros(B, **i32))
    ckpt = hip.ssm_scan_ckpt(T, B, D, N, "cpu").zero_()
    each(hip.ssm_scan_fwd, ["y", "hT", "ckpt"], list(scan) + ["h0"],
         dict(scan, y=z(T, B, D), hT=z(B, D, N), h0=z(B, D, N), ckpt=ckpt, ws=hip.ssm_scan_ws(T, B, D, N, "cpu")))
    grads = dict(du=z(T, B, D), ddt=z(T, B, D), dA=z(D, N), dB=z(T, B, N), dC=z(T, B, N), dD=z(D), dz=z(T, B, D), ddt_bias=z(D), dh0=z(B, D, N),
                 ws=hip.ssm_scan_ws(T, B, D, N, "cpu"))
    each(hip.ssm_scan_bwd, list(grads), list(scan) + ["dy", "ckpt", "dhT"], dict(scan, **grads, dy=z(T, B, D), ckpt=ckpt, dhT=z(B, D, N)))
    each(hip.ssm_step, ["y", "h"], ["u", "dt", "A", "Bm", "Cm", "D", "z", "dt_bias", "reset"],
         dict(u=z(B, D), dt=z(B, D), A=z(D, N), Bm=z(B, N), Cm=z(B, N), h=z(B, D, N), y=z(B, D), D=z(D), z=z(B, D), dt_bias=z(D),
              reset=torch.zeros(B, **u8)))
