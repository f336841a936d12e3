"""The state-space kernels against the formulas in 64 bits (ssm_ref): sizes that divide nothing, episode resets, padding full
of NaN, strided views, both types, missing options, cut sequences, single steps, streams and graphs."""
import pytest
import torch

import ssm_ref
from distributed_rl_amd.ops import hip as H
from distributed_rl_amd.ops import oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    H.native.hip()


class Gen:
    def __init__(self, seed):
        self.g = torch.Generator().manual_seed(seed)

    def n(self, *shape, dtype=F32, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=self.g) * scale + shift).to(dtype).to(DEV)

    def u(self, *shape):
        return torch.rand(*shape, generator=self.g).to(DEV)


def like(*ts):
    """Outputs full of NaN: what is not written shows."""
    return [torch.full(t.shape, float("nan"), dtype=t.dtype, device=t.device) for t in ts]


# ---- layer norm ---------------------------------------------------------------------------------------------------------
def run_norm(v, eps=1e-5):
    (y, dx), mean, rstd = like(v["x"], v["x"]), torch.empty(len(v["x"]), device=DEV), torch.empty(len(v["x"]), device=DEV)
    dw, db = like(v["w"], v["w"])
    H.layer_norm_fwd(v["x"], v["w"], v["b"], y, mean=mean, rstd=rstd, eps=eps)
    H.layer_norm_bwd(v["dy"], v["x"], v["w"], mean, rstd, dx, dw, db if v["b"] is not None else None, H.layer_norm_ws(*v["x"].shape, DEV))
    out = dict(y=y, dx=dx, mean=mean, rstd=rstd, dw=dw)
    return dict(out, db=db) if v["b"] is not None else out


def check_norm(v, eps=1e-5):
    got = run_norm(v, eps)
    w = ssm_ref.f64(v)
    ref, mag = ssm_ref.norm(w, eps), ssm_ref.norm(w, eps, mag=True)
    # a sum over a row: at most 64 terms in one register, then a tree of at most 2^10 of them: 74 roundings; three such
    # sums stand behind dx, and 16 single operations. The sums over rows add at most one rounding for each row.
    for k in got:
        ssm_ref.close(got[k], ref[k], mag[k], 3 * 74 + 16 + (len(v["x"]) if k in ("dw", "db") else 0), k)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("M,D", [(1, 1), (3, 2), (1, 512), (5, 63), (4, 64), (7, 100), (257, 8), (33, 513), (9, 1024), (6, 1032), (5, 3136),
                                 (2, 4099), (3, 8192), (2, 16384), (1030, 40),
                                 (70, 20), (35, 29), (41, 70), (37, 93), (19, 100), (21, 130), (23, 185), (9, 270), (11, 381), (5, 600), (3, 765)])
def test_norm(M, D, dtype):
    g = Gen(M * 31 + D)
    check_norm(dict(x=g.n(M, D, dtype=dtype, scale=2.0, shift=0.7), w=g.n(D, shift=1.0), b=g.n(D), dy=g.n(M, D, dtype=dtype)))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_norm_strided_rows_without_bias_far_from_zero(dtype):
    g = Gen(3)
    wide = g.n(21, 3 * 96 + 5, dtype=dtype, shift=30.0)
    check_norm(dict(x=wide[:, 3:99], w=g.n(96), b=None, dy=g.n(96, 21, dtype=dtype).t().contiguous()))
    check_norm(dict(x=wide[:, 8:104], w=g.n(96), b=g.n(96), dy=wide[:, 104:200]))
    row = g.n(1, 96, dtype=dtype)
    check_norm(dict(x=row.expand(5, 96), w=g.n(96), b=None, dy=row.expand(5, 96)))


def test_norm_constant_rows_and_one_column():
    g = Gen(4)
    check_norm(dict(x=torch.full((3, 40), 2.5, device=DEV), w=g.n(40), b=g.n(40), dy=g.n(3, 40)))
    check_norm(dict(x=g.n(4, 1), w=g.n(1), b=g.n(1), dy=g.n(4, 1)))


# ---- short convolution --------------------------------------------------------------------------------------------------
def conv_case(T, B, D, W, dtype, seed=0, reset=0.2, ragged=True, state=True, bias=True, dstate=True, nan=True):
    g = Gen(seed + T * 7 + B * 3 + D + W)
    v = dict(x=g.n(T, B, D, dtype=dtype), w=g.n(D, W, scale=0.6), bias=g.n(D, scale=0.3) if bias else None,
             state_in=g.n(B, W - 1, D, dtype=dtype) if state else None, dy=g.n(T, B, D, dtype=dtype),
             dstate_out=g.n(B, W - 1, D, dtype=dtype) if dstate else None,
             reset=(g.u(T, B) < reset).to(torch.uint8) if reset else None, lengths=None)
    if ragged:
        n = (g.u(B) * (T + 1)).int().clamp(max=T)
        n[:1], n[1:2] = T, 0
        v["lengths"] = n
        if nan:
            dead = torch.arange(T, device=DEV)[:, None] >= n[None]
            v["x"][dead] = float("nan")
            v["dy"][dead] = float("inf")
    return v


def run_conv(v, silu=True):
    T, B, D = v["x"].shape
    W = v["w"].shape[1]
    y, dx = (torch.full((T, B, D), float("nan"), dtype=v["x"].dtype, device=DEV) for _ in range(2))
    so, dsi = (torch.full((B, W - 1, D), float("nan"), dtype=v["x"].dtype, device=DEV) for _ in range(2))
    dw, db = like(v["w"], v["w"][:, 0])
    H.short_conv_fwd(v["x"], v["w"], v["bias"], y, state_in=v["state_in"], state_out=so, reset=v["reset"], lengths=v["lengths"], silu=silu)
    H.short_conv_bwd(v["dy"], v["x"], v["w"], v["bias"], dx, dw, db if v["bias"] is not None else None, H.short_conv_ws(T, B, D, W, DEV),
                     state_in=v["state_in"], dstate_in=dsi, dstate_out=v["dstate_out"], reset=v["reset"], lengths=v["lengths"], silu=silu)
    out = dict(y=y, state_out=so, dx=dx, dw=dw, dstate_in=dsi)
    return dict(out, db=db) if v["bias"] is not None else out


def check_conv(v, silu=True):
    got = run_conv(v, silu)
    w = ssm_ref.f64(v)
    w["x"], w["dy"] = torch.nan_to_num(w["x"], 0, 0, 0), torch.nan_to_num(w["dy"], 0, 0, 0)
    ref, mag = ssm_ref.conv(w, silu), ssm_ref.conv(w, silu, mag=True)
    T, B, _ = v["x"].shape
    for k in got:    # W + 1 terms, 16 roundings of the sigmoid and its products, W more sums; one for every summed step
        ssm_ref.close(got[k], ref[k], mag[k], 32 + (T * B if k in ("dw", "db") else 0), k)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("T,B,D,W", [(1, 1, 1, 4), (1, 3, 5, 2), (2, 4, 64, 4), (3, 2, 16, 4), (15, 3, 7, 3), (16, 2, 256, 4), (17, 5, 8, 4),
                                     (31, 3, 130, 2), (33, 2, 264, 3), (65, 4, 40, 4), (4, 3, 2, 4), (9, 3, 3, 2), (40, 2, 515, 3), (19, 2, 1027, 4)])
def test_conv(T, B, D, W, dtype):
    check_conv(conv_case(T, B, D, W, dtype))


@pytest.mark.parametrize("kw", [dict(reset=0), dict(reset=1.0), dict(ragged=False), dict(state=False, dstate=False), dict(bias=False),
                                dict(reset=0, ragged=False, state=False, bias=False, dstate=False)])
def test_conv_options(kw):
    check_conv(conv_case(37, 4, 24, 4, F32, **kw))
    check_conv(conv_case(37, 4, 24, 3, BF, **kw), silu=False)


def test_conv_of_views():
    v = conv_case(20, 3, 48, 4, BF, ragged=False)
    g = Gen(9)
    wide = g.n(3, 20, 2 * 48, dtype=BF)
    v["x"], v["dy"] = wide.transpose(0, 1)[..., :48], wide.transpose(0, 1)[..., 48:]
    check_conv(v)
    odd = g.n(20, 3, 101, dtype=BF)
    v["x"], v["dy"] = odd[..., 1:49], odd[..., 52:100]
    check_conv(v)
    a = run_conv(v)
    buf = torch.full((20, 3, 96), 7.0, dtype=BF, device=DEV)          # an output that is a slice: the rest stays
    H.short_conv_fwd(v["x"], v["w"], v["bias"], buf[..., 48:], state_in=v["state_in"], reset=v["reset"])
    assert torch.equal(buf[..., 48:], a["y"]) and bool((buf[..., :48] == 7).all())


@pytest.mark.parametrize("dtype", [F32, BF])
def test_conv_in_pieces_and_in_steps_is_the_whole(dtype):
    v = conv_case(24, 3, 40, 4, dtype, ragged=False)
    whole = run_conv(v)
    st = v["state_in"].clone()
    for a, b in ((0, 1), (1, 3), (3, 20), (20, 24)):
        y, so = like(v["x"][a:b], st)
        H.short_conv_fwd(v["x"][a:b], v["w"], v["bias"], y, state_in=st, state_out=so, reset=v["reset"][a:b])
        assert torch.equal(y, whole["y"][a:b])
        st = so
    assert torch.equal(st, whole["state_out"])
    st = v["state_in"].clone()
    for t in range(24):
        y, = like(v["x"][0])
        H.short_conv_step(v["x"][t], v["w"], v["bias"], st, y, reset=v["reset"][t])
        assert torch.equal(y, whole["y"][t])
    assert torch.equal(st, whole["state_out"])


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("D", [1, 3, 7, 510, 1025])
def test_conv_writes_nothing_beside_its_rows(D, dtype):
    T, B, W, g = 21, 3, 4, Gen(D)
    x, w, dy = g.n(T, B, D + 5, dtype=dtype)[..., 2:D + 2], g.n(D, W), g.n(T, B, D, dtype=dtype)
    y, dx = (torch.full((T, B, D + 7), 7.0, dtype=dtype, device=DEV) for _ in range(2))
    dw, ref, rx = torch.empty_like(w), torch.empty_like(dy), torch.empty_like(dy)
    ws = H.short_conv_ws(T, B, D, W, DEV)
    H.short_conv_fwd(x, w, None, y[..., 3:D + 3])
    H.short_conv_bwd(dy, x, w, None, dx[..., 3:D + 3], dw, None, ws)
    H.short_conv_fwd(x.contiguous(), w, None, ref)
    H.short_conv_bwd(dy, x.contiguous(), w, None, rx, dw, None, ws)
    for got, want in ((y, ref), (dx, rx)):
        assert torch.equal(got[..., 3:D + 3], want)
        assert bool((got[..., :3] == 7).all()) and bool((got[..., D + 3:] == 7).all())


@pytest.mark.parametrize("B,D,W", [(1, 1, 2), (5, 33, 3), (3, 1024, 4), (257, 40, 4), (150, 257, 4), (3, 2, 2)])
def test_conv_step_strided(B, D, W):
    g = Gen(B + D)
    wide = g.n(B, 2 * D + 3, dtype=BF)
    x, w, st = wide[:, 1:D + 1], g.n(D, W), g.n(B, W - 1, D, dtype=BF)
    y, ref = torch.empty(B, D, dtype=BF, device=DEV), st.clone()
    yr, = like(y[None])
    H.short_conv_fwd(x[None], w, None, yr, state_in=ref, silu=False)
    H.short_conv_step(x, w, None, st, y, silu=False)
    assert torch.equal(y, yr[0]) and torch.equal(st, torch.cat([ref[:, 1:], x[:, None]], 1))


# ---- selective scan -----------------------------------------------------------------------------------------------------
def scan_case(T, B, D, N, dtype, seed=0, reset=0.1, ragged=True, opt=True, shift=-2.0, scale=0.7):
    g = Gen(seed + T * 5 + B * 3 + D + N)
    v = dict(u=g.n(T, B, D, dtype=dtype), dt=g.n(T, B, D, dtype=dtype, scale=scale, shift=shift), A=-g.u(D, N) * 2 - 0.05,
             Bm=g.n(T, B, N, dtype=dtype), Cm=g.n(T, B, N, dtype=dtype), dy=g.n(T, B, D, dtype=dtype),
             reset=(g.u(T, B) < reset).to(torch.uint8) if reset else None, lengths=None)
    for k, t in (("D", g.n(D)), ("z", g.n(T, B, D, dtype=dtype)), ("dt_bias", g.n(D, scale=0.3)), ("h0", g.n(B, D, N)), ("dhT", g.n(B, D, N))):
        v[k] = t if opt is True or opt and k in opt else None
    if ragged:
        n = (g.u(B) * (T + 1)).int().clamp(max=T)
        n[:1], n[1:2], n[2:3] = T, 0, 1
        v["lengths"] = n
        dead = torch.arange(T, device=DEV)[:, None] >= n[None]
        for k, bad in (("u", "nan"), ("dt", "nan"), ("Bm", "inf"), ("Cm", "nan"), ("dy", "inf"), ("z", "nan")):
            if v[k] is not None:
                v[k][dead] = float(bad)
    return v


def run_scan(v, softplus=True, ws=None):
    T, B, D = v["u"].shape
    N = v["A"].shape[1]
    typ = v["u"].dtype
    nan = lambda *s, t=F32: torch.full(s, float("nan"), dtype=t, device=DEV)        # noqa: E731
    o = dict(y=nan(T, B, D, t=typ), hT=nan(B, D, N), du=nan(T, B, D, t=typ), ddt=nan(T, B, D, t=typ), dB=nan(T, B, N, t=typ),
             dC=nan(T, B, N, t=typ), dA=nan(D, N), dh0=nan(B, D, N))
    if v["z"] is not None:
        o["dz"] = nan(T, B, D, t=typ)
    if v["D"] is not None:
        o["dD"] = nan(D)
    if v["dt_bias"] is not None:
        o["ddt_bias"] = nan(D)
    ws = H.ssm_scan_ws(T, B, D, N, DEV).fill_(float("nan")) if ws is None else ws
    ckpt = H.ssm_scan_ckpt(T, B, D, N, DEV).fill_(float("nan"))
    kw = dict(D=v["D"], z=v["z"], dt_bias=v["dt_bias"], reset=v["reset"], lengths=v["lengths"], softplus=softplus)
    H.ssm_scan_fwd(v["u"], v["dt"], v["A"], v["Bm"], v["Cm"], o["y"], ws, h0=v["h0"], hT=o["hT"], ckpt=ckpt, **kw)
    H.ssm_scan_bwd(v["dy"], v["u"], v["dt"], v["A"], v["Bm"], v["Cm"], ckpt, o["du"], o["ddt"], o["dA"], o["dB"], o["dC"], ws,
                   dD=o.get("dD"), dz=o.get("dz"), ddt_bias=o.get("ddt_bias"), dhT=v["dhT"], dh0=o["dh0"], **kw)
    return o


def clean(v):
    return {k: (torch.nan_to_num(x, 0, 0, 0) if torch.is_tensor(x) and x.dtype == torch.float64 else x) for k, x in ssm_ref.f64(v).items()}


def check_scan(v, softplus=True):
    got = run_scan(v, softplus)
    w = clean(v)
    ref, mag = ssm_ref.scan(w, softplus), ssm_ref.scan(w, softplus, mag=True)
    for k in got:
        ssm_ref.close(got[k], ref[k], mag[k], ssm_ref.scan_roundings(w, k not in ("y", "hT"), softplus), k)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("T,B,D,N", [(1, 1, 1, 1), (1, 3, 17, 16), (2, 4, 16, 4), (15, 3, 33, 5), (16, 3, 64, 16), (17, 4, 20, 8), (33, 3, 65, 16),
                                     (40, 2, 130, 9), (50, 3, 24, 17), (20, 3, 40, 32), (37, 2, 18, 33), (35, 3, 70, 64), (70, 5, 96, 16)])
def test_scan(T, B, D, N, dtype):
    check_scan(scan_case(T, B, D, N, dtype))


@pytest.mark.parametrize("kw", [dict(reset=0), dict(reset=1.0), dict(ragged=False), dict(opt=False), dict(opt=("z",)), dict(opt=("D",)),
                                dict(opt=("dt_bias", "h0")), dict(reset=0, ragged=False, opt=False)])
@pytest.mark.parametrize("N", [6, 16, 40])
def test_scan_options(kw, N):
    check_scan(scan_case(37, 4, 24, N, F32, **kw))
    check_scan(scan_case(21, 4, 24, N, BF, **kw))


def test_scan_step_sizes_as_given_and_extreme_ones():
    check_scan(scan_case(19, 3, 20, 16, F32, shift=0.3, scale=0.2), softplus=False)             # growing and shrinking states
    check_scan(scan_case(9, 3, 20, 16, F32, shift=15.0, scale=8.0))                             # decays down to nothing
    check_scan(scan_case(9, 3, 20, 16, F32, shift=-60.0, scale=20.0))                           # steps down to nothing
    v = scan_case(20, 3, 20, 16, F32)
    v["A"].zero_()                                                                              # a plain sum
    check_scan(v)


def test_scan_rows_without_a_step():
    v = scan_case(20, 3, 20, 16, F32, ragged=False)
    v["lengths"] = torch.zeros(3, dtype=torch.int32, device=DEV)
    got = run_scan(v)
    assert torch.equal(got["hT"], v["h0"]) and torch.equal(got["dh0"], v["dhT"])
    for k in ("y", "du", "ddt", "dz", "dB", "dC", "dA", "dD", "ddt_bias"):
        assert bool((got[k] == 0).all()), k
    v["lengths"] = torch.tensor([100, -5, 20], dtype=torch.int32, device=DEV)                   # beyond the batch: cut to it
    a = run_scan(v)
    v["lengths"] = torch.tensor([20, 0, 20], dtype=torch.int32, device=DEV)
    b = run_scan(v)
    assert all(torch.equal(a[k], b[k]) for k in a)


@pytest.mark.parametrize("T,B,D,N,dtype", [(300, 1, 16, 16, F32), (523, 1, 40, 8, BF), (1100, 2, 17, 5, F32), (260, 1, 64, 40, F32), (701, 1, 33, 3, BF)])
def test_scan_long_and_few_rows(T, B, D, N, dtype):
    check_scan(scan_case(T, B, D, N, dtype, reset=0.004, shift=-4.0, scale=0.3))
    check_scan(scan_case(T, B, D, N, dtype, reset=0, ragged=False, shift=-4.0, scale=0.3))


@pytest.mark.parametrize("T,B,D", [(20, 3, 40), (600, 1, 16)])                              # one segment, and several
def test_scan_state_of_a_finished_episode_is_never_used(T, B, D):
    v = scan_case(T, B, D, 16, F32, ragged=False, reset=0.01, shift=-4.0, scale=0.3)
    v["reset"][0] = 1
    v["h0"].zero_()
    a = run_scan(v)
    v["h0"].fill_(float("nan"))
    b = run_scan(v)
    assert all(torch.equal(a[k], b[k]) for k in a)
    assert bool((b["dh0"] == 0).all())


@pytest.mark.parametrize("B", [255, 256, 257, 300])
def test_scan_padded_rows_around_the_sorted_count(B):
    check_scan(scan_case(18, B, 5, 3, F32))


def test_scan_of_views():
    g = Gen(11)
    T, B, D, N = 25, 3, 40, 16
    v = scan_case(T, B, D, N, BF, ragged=False)
    xz, bc = g.n(B, T, 2 * D + 1, dtype=BF).transpose(0, 1), g.n(T, B, 7 + 2 * N, dtype=BF)
    v.update(u=xz[..., 1:D + 1], z=xz[..., D + 1:], Bm=bc[..., 7:7 + N], Cm=bc[..., 7 + N:], dy=g.n(T, 1, D, dtype=BF).expand(T, B, D))
    check_scan(v)
    a = run_scan(v)
    dxz, dbc = torch.full((T, B, 2 * D), 7.0, dtype=BF, device=DEV), torch.full((B, T, 3 * N), 7.0, dtype=BF, device=DEV).transpose(0, 1)
    ws, ckpt = H.ssm_scan_ws(T, B, D, N, DEV), H.ssm_scan_ckpt(T, B, D, N, DEV)
    kw = dict(D=v["D"], z=v["z"], dt_bias=v["dt_bias"], reset=v["reset"])
    H.ssm_scan_fwd(v["u"], v["dt"], v["A"], v["Bm"], v["Cm"], dxz[..., :D], ws, h0=v["h0"], ckpt=ckpt, **kw)
    assert torch.equal(dxz[..., :D], a["y"]) and bool((dxz[..., D:] == 7).all())
    ddt, dA = torch.empty(T, B, D, dtype=BF, device=DEV), torch.empty(D, N, device=DEV)
    H.ssm_scan_bwd(v["dy"], v["u"], v["dt"], v["A"], v["Bm"], v["Cm"], ckpt, dxz[..., :D], ddt, dA, dbc[..., :N], dbc[..., N:2 * N], ws,
                   dz=dxz[..., D:], dhT=v["dhT"], **kw)
    for k, t in (("du", dxz[..., :D]), ("dz", dxz[..., D:]), ("ddt", ddt), ("dA", dA), ("dB", dbc[..., :N]), ("dC", dbc[..., N:2 * N])):
        assert torch.equal(t, a[k]), k
    assert bool((dbc[..., 2 * N:] == 7).all())


def test_scan_in_pieces_is_the_whole():
    """Burn-in and training window as two calls, the state carried over; and every step by itself."""
    v = scan_case(56, 3, 48, 16, F32, ragged=False)
    w = clean(v)
    ref, mag = ssm_ref.scan(w), ssm_ref.scan(w, mag=True)
    n = ssm_ref.scan_roundings(w, False)
    h, ys = v["h0"], []
    for a, b in ((0, 1), (1, 24), (24, 56)):
        y, hT = torch.empty_like(v["u"][a:b]), torch.empty_like(h)
        H.ssm_scan_fwd(*(v[k][a:b] if k != "A" else v[k] for k in ("u", "dt", "A", "Bm", "Cm")), y, H.ssm_scan_ws(b - a, 3, 48, 16, DEV, train=False),
                       D=v["D"], z=v["z"][a:b], dt_bias=v["dt_bias"], h0=h, hT=hT, reset=v["reset"][a:b])
        h = hT
        ys.append(y)
    ssm_ref.close(torch.cat(ys), ref["y"], mag["y"], n, "y")
    ssm_ref.close(h, ref["hT"], mag["hT"], n, "hT")
    h, ys = v["h0"].clone(), []
    for t in range(56):
        ys.append(torch.empty_like(v["u"][0]))
        H.ssm_step(v["u"][t], v["dt"][t], v["A"], v["Bm"][t], v["Cm"][t], h, ys[-1], D=v["D"], z=v["z"][t], dt_bias=v["dt_bias"], reset=v["reset"][t])
    ssm_ref.close(torch.stack(ys), ref["y"], mag["y"], n, "y by steps")
    ssm_ref.close(h, ref["hT"], mag["hT"], n, "h by steps")


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("B,D,N", [(1, 1, 1), (3, 17, 16), (5, 64, 4), (2, 100, 8), (7, 33, 5), (4, 70, 32), (3, 40, 64), (2, 9, 47), (130, 40, 16)])
def test_step(B, D, N, dtype):
    v = scan_case(1, B, D, N, dtype, ragged=False, reset=0.3)
    for opt in (True, False):
        if not opt:
            v.update(D=None, z=None, dt_bias=None, reset=None)
        w = clean({k: x for k, x in v.items() if k not in ("dy", "dhT")})
        ref, mag = ssm_ref.scan(w), ssm_ref.scan(w, mag=True)
        h, y = v["h0"].clone(), torch.full((B, D), float("nan"), dtype=dtype, device=DEV)
        sl = lambda k: v[k][0] if v[k] is not None else None                        # noqa: E731
        H.ssm_step(sl("u"), sl("dt"), v["A"], sl("Bm"), sl("Cm"), h, y, D=v["D"], z=sl("z"), dt_bias=v["dt_bias"], reset=sl("reset"))
        n = ssm_ref.scan_roundings(w, False)
        ssm_ref.close(y, ref["y"][0], mag["y"][0], n, "y")
        ssm_ref.close(h, ref["hT"], mag["hT"], n, "h")


def test_step_of_views():
    g = Gen(2)
    B, D, N = 5, 24, 16
    wide, bc = g.n(B, 3 * D + 1, dtype=BF), g.n(B, 2 * N + 3, dtype=BF)
    A, h = -g.u(D, N), g.n(B, D, N)
    h2, y, y2 = h.clone(), torch.full((B, 2 * D), 7.0, dtype=BF, device=DEV), torch.empty(B, D, dtype=BF, device=DEV)
    a = (wide[:, 1:D + 1], wide[:, D + 1:2 * D + 1], A, bc[:, 3:3 + N], bc[:, 3 + N:])
    H.ssm_step(*a, h, y[:, :D], z=wide[:, 2 * D + 1:])
    H.ssm_step(*(t.contiguous() for t in a), h2, y2, z=wide[:, 2 * D + 1:].contiguous())
    assert torch.equal(y[:, :D], y2) and torch.equal(h, h2) and bool((y[:, D:] == 7).all())


# ---- steps that are held, states that diverged, factors of a segment that leave the range -------------------------------------
def check_scan_tight(v, softplus=True, w=None):
    """Against bounds that fade as the states do. ``w``: the values in 64 bits, where they are not all finite."""
    got = run_scan(v, softplus)
    w = clean(v) if w is None else w
    ref, tol = ssm_ref.scan(w, softplus), ssm_ref.scan_bounds(w, softplus, cut=w["u"].shape[0] > 112)
    for k in got:
        ssm_ref.within(got[k], ref[k], tol[k], k)
    return got


LOWEST = [float("-inf"), torch.finfo(BF).min, -2.37e38, -129.0]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("low", LOWEST)
@pytest.mark.parametrize("T,B,D,N", [(21, 4, 20, 16), (40, 2, 24, 40), (600, 2, 16, 8)])
def test_scan_holds_its_state_over_steps_of_the_lowest_size(T, B, D, N, low, dtype):
    v = scan_case(T, B, D, N, dtype, reset=0.02)
    held = Gen(T).u(T, B) < 0.3
    v["dt"][held] = low
    w = clean(v)
    w["dt"][held.cpu()] = low                                                       # clean() takes infinities out
    got = check_scan_tight(v, w=w)
    assert bool((got["ddt"][held] == 0).all())


@pytest.mark.parametrize("T,B,D", [(40, 2, 24), (600, 2, 16)])
def test_scan_takes_no_nan_for_a_held_step(T, B, D):
    v = scan_case(T, B, D, 16, F32, reset=0, ragged=False)
    v["dt"][T // 2, 0] = float("nan")
    y = run_scan(v)["y"]
    assert bool(y[T // 2:, 0].isnan().all()) and not bool(y[:T // 2].isnan().any()) and not bool(y[:, 1:].isnan().any())


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("low", LOWEST + [torch.finfo(F32).min])
@pytest.mark.parametrize("B,D,N", [(3, 17, 16), (4, 9, 5), (2, 70, 64)])
def test_step_of_the_lowest_size_leaves_the_state(B, D, N, low, dtype):
    v = scan_case(1, B, D, N, dtype, ragged=False, reset=0)
    h, y = v["h0"].clone(), torch.empty(B, D, dtype=dtype, device=DEV)
    dt = torch.full_like(v["dt"][0], low, dtype=F32).to(dtype)                      # (fp32's lowest value is -inf in bf16)
    H.ssm_step(v["u"][0], dt, v["A"], v["Bm"][0], v["Cm"][0], h, y, D=v["D"], z=v["z"][0], dt_bias=v["dt_bias"])
    assert torch.equal(h, v["h0"])
    w = clean({k: x for k, x in v.items() if k not in ("dy", "dhT")})
    w["dt"] = torch.full_like(w["dt"], low)
    ssm_ref.within(y, ssm_ref.scan(w)["y"][0], ssm_ref.scan_bounds(w)["y"][0], "y")


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("N", [3, 8, 16, 24, 40, 64])
@pytest.mark.parametrize("T,B,D,cuts,at", [(50, 2, 20, (3, 9, 16, 24, 37), 20), (50, 1, 20, (8, 13, 21), 15), (600, 1, 16, (24, 200, 383, 400), 250)])
def test_scan_resets_shield_an_episode_from_one_that_diverged(T, B, D, cuts, at, N, bad):
    """What diverges in the episode of step ``at``, its state or its gradient, leaves every other episode bit for bit alone."""
    v = scan_case(T, B, D, N, F32, reset=0, ragged=False, shift=-4.0, scale=0.3)
    v["reset"] = torch.zeros(T, B, dtype=torch.uint8, device=DEV)
    v["reset"][list(cuts)] = 1
    a, b = max(c for c in cuts if c <= at), min(c for c in cuts if c > at)
    good = run_scan(v)
    for k in ("u", "dy"):
        w = dict(v)
        w[k] = v[k].clone()
        w[k][at] = bad
        got = run_scan(w)
        for n in ("y", "du", "ddt", "dz", "dB", "dC"):
            assert torch.equal(got[n][:a], good[n][:a]), (k, n, "before")
            assert torch.equal(got[n][b:], good[n][b:]), (k, n, "behind")
        assert torch.equal(got["hT"], good["hT"]) and torch.equal(got["dh0"], good["dh0"]), k


@pytest.mark.parametrize("rate,h0", [(1.2, 1e-20), (-1.2, 1e25)])
def test_scan_segment_factors_beyond_the_range(rate, h0):
    """Segments of 600 steps whose exp(A sum of s) leaves the range of fp32, while the state that it stands for does not."""
    v = scan_case(600, 1, 16, 16, F32, reset=0, ragged=False, opt=("h0", "dhT"))
    v["A"].fill_(1.0)
    v["dt"].zero_()
    v["dt"][80:160] = rate                                  # exp(96) over one segment
    v["u"][80:160] = 0
    v["h0"], v["dhT"], v["dy"] = v["h0"] * h0, v["dhT"] * h0, v["dy"] * 1e-20
    check_scan_tight(v, softplus=False)


def test_scan_segment_factors_beyond_the_range_of_an_empty_state():
    v = scan_case(600, 1, 16, 16, F32, reset=0, ragged=False, opt=False)
    v["A"].fill_(1.0)
    v["dt"].fill_(0.01)
    v["dt"][80:320] = 1.2
    v["u"][:320] = 0                                        # no state before step 320, and no gradient from there on
    v["dy"][80:] = 0
    check_scan_tight(v, softplus=False)


@pytest.mark.parametrize("T,B,D,N", [(21, 4, 20, 16), (40, 3, 24, 5), (600, 4, 16, 8)])
def test_scan_decay_rates_of_the_lowest_value(T, B, D, N):
    """A = the lowest value of the type: a state without memory, but held where a row has ended and over steps of size zero."""
    v = scan_case(T, B, D, N, F32, reset=0.02, shift=-1.0)
    v["A"][:, ::2] = torch.finfo(F32).min
    check_scan_tight(v)
    # the gradient of a held step is the lowest value times a state; and -inf times a step of zero is no number
    for low, size in ((torch.finfo(F32).min, float("-inf")), (float("-inf"), 0.0)):
        v["A"][:, ::2], v["dt"][T // 3] = low, size
        w = clean({k: x for k, x in v.items() if k != "dy"})
        w["A"][:, ::2], w["dt"][T // 3] = torch.finfo(F32).min, size
        got, ref, tol = run_scan(v), ssm_ref.scan(w), ssm_ref.scan_bounds(w, cut=T > 112)
        for k in ("y", "hT"):
            ssm_ref.within(got[k], ref[k], tol[k], k)


@pytest.mark.parametrize("N", [16, 5])
def test_step_with_decay_rates_of_the_lowest_value(N):
    v = scan_case(1, 3, 20, N, F32, ragged=False, reset=0)
    for low, size in ((torch.finfo(F32).min, -1.0), (torch.finfo(F32).min, float("-inf")), (float("-inf"), -1.0)):
        v["A"][:, ::2] = low
        dt = torch.full_like(v["dt"][0], size)
        h, y = v["h0"].clone(), torch.empty_like(v["u"][0])
        H.ssm_step(v["u"][0], dt, v["A"], v["Bm"][0], v["Cm"][0], h, y, D=v["D"], z=v["z"][0], dt_bias=v["dt_bias"])
        w = clean({k: x for k, x in v.items() if k not in ("dy", "dhT")})
        w["dt"], w["A"][:, ::2] = torch.full_like(w["dt"], size), torch.finfo(F32).min
        ref, tol = ssm_ref.scan(w), ssm_ref.scan_bounds(w)
        ssm_ref.within(y, ref["y"][0], tol["y"][0], "y")
        ssm_ref.within(h, ref["hT"], tol["hT"], "h")


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("N,reset", [(16, 0), (5, 0.01), (40, 0.01)])
def test_scan_rows_that_end_inside_a_cut_sequence(N, reset, dtype):
    """600 steps of ten short rows are cut into segments of 80: rows that end in the middle of a chunk, around a segment's border,
    with the first step, and never; what is behind is NaN."""
    T, D = 600, 16
    ends = torch.tensor([T, 245, 240, 239, 241, 1, 0, 480, 473, 81], dtype=torch.int32)
    v = scan_case(T, len(ends), D, N, dtype, reset=reset, ragged=False, shift=-4.0, scale=0.3)
    v["lengths"] = ends.to(DEV)
    dead = torch.arange(T, device=DEV)[:, None] >= v["lengths"][None]
    for k in ("u", "dt", "Bm", "Cm", "dy", "z"):
        v[k][dead] = float("nan")
    got = check_scan_tight(v)
    assert torch.equal(got["hT"][6], v["h0"][6]) and torch.equal(got["dh0"][6], v["dhT"][6])
    for k in ("y", "du", "ddt", "dz", "dB", "dC"):
        assert bool((got[k][dead] == 0).all()), k


@pytest.mark.parametrize("T,B,D,N,dtype", [(1100, 2, 17, 5, F32), (523, 1, 40, 8, BF), (260, 1, 64, 40, F32), (120, 3, 70, 16, F32), (90, 2, 33, 24, BF)])
def test_scan_of_long_sequences_within_bounds_that_fade(T, B, D, N, dtype):
    check_scan_tight(scan_case(T, B, D, N, dtype, reset=0.004, shift=-4.0, scale=0.3))
    check_scan_tight(scan_case(T, B, D, N, dtype, reset=0, ragged=False, shift=-4.0, scale=0.3))


# ---- offsets past 32 bits -----------------------------------------------------------------------------------------------
def test_norm_past_32_bits():
    M, D = 150000, 16384                                    # 2.46e9 elements
    x = torch.empty(M, D, dtype=BF, device=DEV)
    x.random_(-8, 9)
    y, w = torch.empty_like(x), torch.ones(D, device=DEV)
    mean, rstd = torch.empty(M, device=DEV), torch.empty(M, device=DEV)
    H.layer_norm_fwd(x, w, None, y, mean=mean, rstd=rstd)
    part = torch.empty(3, D, dtype=BF, device=DEV)
    H.layer_norm_fwd(x[-3:], w, None, part)
    assert torch.equal(y[-3:], part)
    dw = torch.empty(D, device=DEV)
    H.layer_norm_bwd(x, x, w, mean, rstd, y, dw, None, H.layer_norm_ws(M, D, DEV))
    dx = torch.empty_like(part)
    H.layer_norm_bwd(x[-3:], x[-3:], w, mean[-3:], rstd[-3:], dx, dw, None, H.layer_norm_ws(3, D, DEV))
    assert torch.equal(y[-3:], dx)


def test_norm_of_more_rows_than_a_launch_takes():
    M, D = (1 << 21) * 64 + 5, 4
    x = torch.empty(M, D, dtype=BF, device=DEV)
    x.random_(-8, 9)
    y, w, mean, rstd = torch.empty_like(x), torch.ones(D, device=DEV), torch.empty(M, device=DEV), torch.empty(M, device=DEV)
    H.layer_norm_fwd(x, w, None, y, mean=mean, rstd=rstd)
    for cut in (slice(0, 7), slice(M - 9, M)):
        part = [torch.empty_like(x[cut]), torch.empty_like(mean[cut]), torch.empty_like(mean[cut])]
        H.layer_norm_fwd(x[cut], w, None, part[0], mean=part[1], rstd=part[2])
        assert torch.equal(y[cut], part[0]) and torch.equal(mean[cut], part[1]) and torch.equal(rstd[cut], part[2])


def test_conv_and_scan_past_32_bits():
    T, B, D, N = 2100, 1024, 1024, 2                        # 2.2e9 elements a tensor
    g = Gen(0)
    x = torch.empty(T, B, D, dtype=BF, device=DEV)
    x.random_(-2, 3)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    w, dw = g.n(D, 4), torch.empty(D, 4, device=DEV)
    last = x[:, -1:].contiguous()
    p, q = torch.empty_like(last), torch.empty_like(last)
    H.short_conv_fwd(x, w, None, y)
    H.short_conv_fwd(last, w, None, p)
    assert torch.equal(y[:, -1:], p)
    H.short_conv_bwd(x, x, w, None, dx, dw, None, H.short_conv_ws(T, B, D, 4, DEV))
    H.short_conv_bwd(last, last, w, None, q, dw, None, H.short_conv_ws(T, 1, D, 4, DEV))
    assert torch.equal(dx[:, -1:], q)
    A, bc = -g.u(D, N) - 0.5, g.n(T, B, 2 * N, dtype=BF)
    ws, ck = H.ssm_scan_ws(T, B, D, N, DEV), H.ssm_scan_ckpt(T, B, D, N, DEV)
    H.ssm_scan_fwd(x, x, A, bc[..., :N], bc[..., N:], y, ws, ckpt=ck)
    dA, dB, dC = torch.empty(D, N, device=DEV), torch.empty(T, B, N, dtype=BF, device=DEV), torch.empty(T, B, N, dtype=BF, device=DEV)
    ddt = torch.empty_like(x)
    H.ssm_scan_bwd(x, x, x, A, bc[..., :N], bc[..., N:], ck, dx, ddt, dA, dB, dC, ws)
    # the last row by itself: cut into segments there, so equal up to rounding (2 100 steps, decays of at most exp(-0.06))
    bl = bc[:, -1:].contiguous()
    o = [torch.empty_like(last) for _ in range(3)]
    oB, oC = torch.empty(T, 1, N, dtype=BF, device=DEV), torch.empty(T, 1, N, dtype=BF, device=DEV)
    ws, ck = H.ssm_scan_ws(T, 1, D, N, DEV), H.ssm_scan_ckpt(T, 1, D, N, DEV)
    H.ssm_scan_fwd(last, last, A, bl[..., :N], bl[..., N:], o[0], ws, ckpt=ck)
    H.ssm_scan_bwd(last, last, last, A, bl[..., :N], bl[..., N:], ck, o[1], o[2], dA, oB, oC, ws)
    for a, b in ((y[:, -1:], o[0]), (dx[:, -1:], o[1]), (ddt[:, -1:], o[2]), (dB[:, -1:], oB), (dC[:, -1:], oC)):
        a, b = a.double(), b.double()
        assert float((a - b).norm() / b.norm()) < 2.0 ** -8                # each is rounded to bf16 once: 2^-8 between the two


def test_scan_of_one_step_of_many_rows():
    # the stride of the one step is 1.3e8 elements: offsets inside a chunk must not count it
    B, D = 65535, 2048
    g = Gen(0)
    u = torch.empty(1, B, D, dtype=BF, device=DEV)
    u.random_(-2, 3)
    A, bc = -g.u(D, 1) - 0.5, g.n(1, B, 2, dtype=BF)
    y, hT, ws = torch.empty_like(u), torch.empty(B, D, 1, device=DEV), H.ssm_scan_ws(1, B, D, 1, DEV)
    ck = H.ssm_scan_ckpt(1, B, D, 1, DEV)
    o = [torch.empty_like(u) for _ in range(2)] + [torch.empty(D, 1, device=DEV)] + [torch.empty(1, B, 1, dtype=BF, device=DEV) for _ in range(2)]
    H.ssm_scan_fwd(u, u, A, bc[..., :1], bc[..., 1:], y, ws, hT=hT, ckpt=ck)
    H.ssm_scan_bwd(u, u, u, A, bc[..., :1], bc[..., 1:], ck, *o, ws)
    for cut in (slice(0, 3), slice(B - 3, B)):
        v, b = u[:, cut].contiguous(), bc[:, cut].contiguous()
        p, q = torch.empty_like(v), [torch.empty_like(v) for _ in range(2)] + [o[2].clone()] + [torch.empty(1, 3, 1, dtype=BF, device=DEV) for _ in range(2)]
        h, w, c = torch.empty(3, D, 1, device=DEV), H.ssm_scan_ws(1, 3, D, 1, DEV), H.ssm_scan_ckpt(1, 3, D, 1, DEV)
        H.ssm_scan_fwd(v, v, A, b[..., :1], b[..., 1:], p, w, hT=h, ckpt=c)
        H.ssm_scan_bwd(v, v, v, A, b[..., :1], b[..., 1:], c, *q, w)
        assert torch.equal(y[:, cut], p) and torch.equal(hT[cut], h)
        assert torch.equal(o[0][:, cut], q[0]) and torch.equal(o[1][:, cut], q[1]) and torch.equal(o[3][:, cut], q[3]) and torch.equal(o[4][:, cut], q[4])


def test_gradients_of_more_elements_than_a_launch_takes():
    # 1.1e9 elements of dB and dC. Every step starts an episode, so dB = dy C s u and dC = dy s u B by themselves.
    T, N = (1 << 23) + 70, 64
    g = Gen(0)
    u, dy = g.n(T, 1, 1, dtype=BF), g.n(T, 1, 1, dtype=BF)
    bc = torch.empty(T, 1, 2 * N, dtype=BF, device=DEV)
    bc.random_(-2, 3)
    dt, A, one = torch.full_like(u, 0.5), -torch.ones(1, N, device=DEV), torch.ones(T, 1, dtype=torch.uint8, device=DEV)
    y, ws, ck = torch.empty_like(u), H.ssm_scan_ws(T, 1, 1, N, DEV), H.ssm_scan_ckpt(T, 1, 1, N, DEV)
    o = [torch.empty_like(u) for _ in range(2)] + [torch.empty(1, N, device=DEV)] + [torch.empty(T, 1, N, dtype=BF, device=DEV) for _ in range(2)]
    H.ssm_scan_fwd(u, dt, A, bc[..., :N], bc[..., N:], y, ws, reset=one, softplus=False, ckpt=ck)
    H.ssm_scan_bwd(dy, u, dt, A, bc[..., :N], bc[..., N:], ck, *o, ws, reset=one, softplus=False)
    for cut in (slice(0, 1000), slice(T - 1000, T)):
        f = (dy[cut].double() * 0.5 * u[cut].double())
        for got, x in ((o[3], bc[cut, :, N:]), (o[4], bc[cut, :, :N])):
            want = f * x.double()
            assert bool(((got[cut].double() - want).abs() <= want.abs() * 2.0 ** -8 * 1.01).all())      # one rounding to bf16


def test_steps_of_more_channels_than_a_launch_takes():
    B, D, N = 70000, 2048, 33                               # 1.4e8 channels of 64 lanes
    g = Gen(0)
    u = torch.empty(B, D, dtype=BF, device=DEV)
    u.random_(-2, 3)
    A, bc, y, h = -g.u(D, N), g.n(B, 2 * N, dtype=BF), torch.empty_like(u), torch.ones(B, D, N, device=DEV)
    H.ssm_step(u, u, A, bc[:, :N], bc[:, N:], h, y)
    for cut in (slice(0, 2), slice(B - 2, B)):
        p, k = torch.empty_like(u[cut]), torch.ones(2, D, N, device=DEV)
        H.ssm_step(u[cut], u[cut], A, bc[cut, :N], bc[cut, N:], k, p)
        assert torch.equal(p, y[cut]) and torch.equal(k, h[cut])
    del u, y, h
    B, D, W = 2100000, 1025, 2                              # 2.2e9 channels, one a thread
    x, s = torch.empty(B, D, dtype=BF, device=DEV), torch.empty(B, 1, D, dtype=BF, device=DEV)
    x.random_(-2, 3); s.fill_(0.5)
    w, y = g.n(D, W), torch.empty_like(x)
    H.short_conv_step(x, w, None, s, y)
    for cut in (slice(0, 2), slice(B - 2, B)):
        p, k = torch.empty_like(x[cut]), torch.full((2, 1, D), 0.5, dtype=BF, device=DEV)
        H.short_conv_step(x[cut], w, None, k, p)
        assert torch.equal(p, y[cut]) and torch.equal(k, s[cut])


# ---- same inputs, same bits; streams; graphs ----------------------------------------------------------------------------
def test_results_do_not_change_from_call_to_call():
    for v in (scan_case(70, 5, 96, 16, BF), scan_case(523, 1, 40, 8, F32)):
        a, b = run_scan(v), run_scan(v)
        assert all(torch.equal(a[k], b[k]) for k in a)
    v = conv_case(65, 4, 264, 4, F32)
    a, b = run_conv(v), run_conv(v)
    assert all(torch.equal(a[k], b[k]) for k in a)
    g = Gen(0)
    v = dict(x=g.n(1030, 40), w=g.n(40), b=g.n(40), dy=g.n(1030, 40))
    a, b = run_norm(v), run_norm(v)
    assert all(torch.equal(a[k], b[k]) for k in a)


def test_two_streams_at_once():
    va, vb = scan_case(300, 2, 64, 16, F32, seed=1), scan_case(300, 2, 64, 16, F32, seed=2)
    ra, rb = run_scan(va), run_scan(vb)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(sa):
            a = run_scan(va)
        with torch.cuda.stream(sb):
            b = run_scan(vb)
        torch.cuda.synchronize()
        assert all(torch.equal(a[k], ra[k]) for k in a) and all(torch.equal(b[k], rb[k]) for k in b)


def core(v, s):
    """One residual block of the core, forward and backward, the way an engine strings the operators together: norm -> short
    convolution -> scan -> y + x, into the buffers of ``s``."""
    T, B, D = v["x"].shape
    flat = lambda t: t.view(T * B, D)                                              # noqa: E731
    H.layer_norm_fwd(flat(v["x"]), v["nw"], v["nb"], flat(s["n"]), mean=s["mean"], rstd=s["rstd"])
    H.short_conv_fwd(s["n"], v["w"], v["bias"], s["c"], state_in=v["cs"], state_out=s["cs"], reset=v["reset"], lengths=v["lengths"])
    kw = dict(D=v["D"], z=v["z"], dt_bias=v["dt_bias"], reset=v["reset"], lengths=v["lengths"])
    H.ssm_scan_fwd(s["c"], v["dt"], v["A"], v["Bm"], v["Cm"], s["y"], s["ws"], h0=v["h0"], hT=s["hT"], ckpt=s["ckpt"], **kw)
    H.ssm_scan_bwd(v["dy"], s["c"], v["dt"], v["A"], v["Bm"], v["Cm"], s["ckpt"], s["dc"], s["ddt"], s["dA"], s["dB"], s["dC"], s["ws"], dD=s["dD"],
                   dz=s["dz"], ddt_bias=s["ddt_bias"], dh0=s["dh0"], **kw)
    H.short_conv_bwd(s["dc"], s["n"], v["w"], v["bias"], s["dn"], s["dw"], s["db"], s["cws"], state_in=v["cs"], dstate_in=s["dcs"],
                     reset=v["reset"], lengths=v["lengths"])
    H.layer_norm_bwd(flat(s["dn"]), flat(v["x"]), v["nw"], s["mean"], s["rstd"], flat(s["dx"]), s["dnw"], s["dnb"], s["nws"])


def core_case(T=40, B=4, D=72, N=16, W=4, seed=0):
    g = Gen(seed)
    v = scan_case(T, B, D, N, F32, seed=seed, ragged=False)
    v.update(x=g.n(T, B, D), nw=g.n(D, shift=1.0, scale=0.2), nb=g.n(D, scale=0.2), w=g.n(D, W, scale=0.5), bias=g.n(D, scale=0.1), cs=g.n(B, W - 1, D))
    v["lengths"] = torch.tensor([T, 0, 1, T - 7][:B], dtype=torch.int32, device=DEV)
    e = lambda *s: torch.full(s, float("nan"), device=DEV)                          # noqa: E731
    s = {k: e(T, B, D) for k in ("n", "c", "y", "dc", "ddt", "dz", "dn", "dx")}
    s.update(mean=e(T * B), rstd=e(T * B), cs=e(B, W - 1, D), hT=e(B, D, N), dA=e(D, N), dB=e(T, B, N), dC=e(T, B, N), dD=e(D), ddt_bias=e(D),
             dh0=e(B, D, N), dw=e(D, W), db=e(D), dcs=e(B, W - 1, D), dnw=e(D), dnb=e(D), ws=H.ssm_scan_ws(T, B, D, N, DEV),
             ckpt=H.ssm_scan_ckpt(T, B, D, N, DEV), cws=H.short_conv_ws(T, B, D, W, DEV), nws=H.layer_norm_ws(T * B, D, DEV))
    return v, s


def test_the_operators_together_against_autograd_in_64_bits():
    v, s = core_case()
    core(v, s)
    p = {k: t.detach().cpu().double().requires_grad_() for k, t in v.items() if t is not None and t.is_floating_point() and k not in ("dy", "dhT", "u")}
    reset, lengths = v["reset"].cpu(), v["lengths"].cpu()
    n = oracle.layer_norm(p["x"], p["nw"], p["nb"])
    c, cs = oracle.short_conv(n, p["w"], p["bias"], p["cs"], reset, lengths)
    y, hT = oracle.ssm_scan(c, p["dt"], p["A"], p["Bm"], p["Cm"], p["D"], p["z"], p["dt_bias"], p["h0"], reset, lengths)
    (y * v["dy"].cpu().double()).sum().backward()
    pairs = dict(y=y, hT=hT, cs=cs, dx=p["x"].grad, dnw=p["nw"].grad, dnb=p["nb"].grad, dw=p["w"].grad, db=p["bias"].grad, dcs=p["cs"].grad,
                 ddt=p["dt"].grad, dz=p["z"].grad, dA=p["A"].grad, dB=p["Bm"].grad, dC=p["Cm"].grad, dD=p["D"].grad, ddt_bias=p["dt_bias"].grad,
                 dh0=p["h0"].grad)
    for k, ref in pairs.items():
        # the longest chain: 2 x 40 steps of (14 + exponents) roundings and sums over 160 rows; 2e-4 = 3 400 half steps
        got, ref = s[k].cpu().double(), ref.detach()
        assert float((got - ref).norm() / ref.norm()) < 2e-4, k


def test_the_operators_together_acting_step_by_step():
    """Acting one step at a time gives what the learner's sequence form gives."""
    v, s = core_case()
    v["lengths"] = None
    core(v, s)
    T, B, D = v["x"].shape
    h, cs = v["h0"].clone(), v["cs"].clone()
    for t in range(T):
        n, c, y = like(v["x"][0], v["x"][0], v["x"][0])
        H.layer_norm_fwd(v["x"][t], v["nw"], v["nb"], n)
        H.short_conv_step(n, v["w"], v["bias"], cs, c, reset=v["reset"][t])
        H.ssm_step(c, v["dt"][t], v["A"], v["Bm"][t], v["Cm"][t], h, y, D=v["D"], z=v["z"][t], dt_bias=v["dt_bias"], reset=v["reset"][t])
        assert torch.equal(n, s["n"][t]) and torch.equal(c, s["c"][t])
        torch.testing.assert_close(y, s["y"][t], rtol=1e-4, atol=1e-4)
    assert torch.equal(cs, s["cs"])
    torch.testing.assert_close(h, s["hT"], rtol=1e-4, atol=1e-4)


def test_captured_and_replayed_on_new_inputs():
    """Two graphs with a workspace each; every replay, with eager calls and synchronisations in between, is the eager result."""
    sets = [core_case(T=300, B=2, D=40, seed=k) for k in (1, 2)]
    graphs = []
    for v, s in sets:
        core(v, s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            core(v, s)
        graphs.append(g)
    for k in range(3):
        fresh = [core_case(T=300, B=2, D=40, seed=10 + 2 * k + i) for i in range(2)]
        for (v, s), (w, _) in zip(sets, fresh):
            for n, t in v.items():
                if t is not None:
                    t.copy_(w[n])
        for g in graphs:
            g.replay()
        for (v, s), (w, e) in zip(sets, fresh):
            core(w, e)
            torch.cuda.synchronize()
            for n in e:
                if n not in ("ws", "ckpt", "cws", "nws"):
                    assert torch.equal(e[n], s[n]), n


# ---- refusals on the GPU ------------------------------------------------------------------------------------------------
def test_tensors_of_another_device_than_the_current_one_are_refused(monkeypatch):
    x, w = torch.zeros(2, 8, device=DEV), torch.ones(8, device=DEV)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(ValueError, match="current device"):
        H.layer_norm_fwd(x, w, w, torch.empty_like(x))
    with pytest.raises(ValueError, match="current device"):
        H.short_conv_step(x, torch.zeros(8, 4, device=DEV), w, torch.zeros(2, 3, 8, device=DEV), torch.empty_like(x))
    with pytest.raises(ValueError, match="current device"):
        H.ssm_step(x, x.clone(), torch.zeros(8, 2, device=DEV), x[:, :2], x[:, 2:4], torch.zeros(2, 8, 2, device=DEV), torch.empty_like(x))


def test_refusals():
    g = Gen(0)
    T, B, D, N = 5, 2, 8, 4
    v = scan_case(T, B, D, N, F32, ragged=False)
    y, ws = torch.zeros_like(v["u"]), H.ssm_scan_ws(T, B, D, N, DEV)
    ok = dict(u=v["u"], dt=v["dt"], A=v["A"], Bm=v["Bm"], Cm=v["Cm"], y=y, ws=ws)

    def bad(exc, **kw):
        with pytest.raises(exc):
            H.ssm_scan_fwd(**{**ok, **kw})

    H.ssm_scan_fwd(**ok)
    bad(TypeError, dt=v["dt"].to(BF))
    bad(TypeError, u=v["u"].half(), dt=v["dt"].half())
    bad(TypeError, A=v["A"].double())
    bad(TypeError, Bm=v["Bm"].cpu())
    bad(TypeError, reset=torch.zeros(T, B, dtype=torch.bool, device=DEV))
    bad(TypeError, lengths=torch.zeros(B, dtype=torch.int64, device=DEV))
    bad(ValueError, A=v["A"][:, :3])
    bad(ValueError, Cm=v["Cm"][:4])
    bad(ValueError, lengths=torch.zeros(B + 1, dtype=torch.int32, device=DEV))
    bad(ValueError, y=v["u"])
    bad(ValueError, hT=v["h0"], h0=v["h0"])
    bad(ValueError, dt=v["dt"].transpose(0, 2).contiguous().transpose(0, 2))
    bad(ValueError, y=torch.zeros(1, B, D, device=DEV).expand(T, B, D))
    bad(ValueError, ckpt=torch.zeros(2, B, D, N, device=DEV))
    grads = dict(du=y.clone(), ddt=y.clone(), dA=torch.zeros(D, N, device=DEV), dB=torch.zeros(T, B, N, device=DEV), dC=torch.zeros(T, B, N, device=DEV))
    with pytest.raises(RuntimeError, match="-2"):
        H.ssm_scan_bwd(v["dy"], v["u"], v["dt"], v["A"], v["Bm"], v["Cm"], H.ssm_scan_ckpt(T, B, D, N, DEV), ws=torch.zeros(3, device=DEV), **grads)
    with pytest.raises(ValueError):
        H.ssm_scan_ws(5, 2, 8, 65, DEV)
    x = g.n(6, 8)
    with pytest.raises(RuntimeError, match="-2"):
        H.layer_norm_bwd(x, x.clone(), g.n(8), g.n(6), g.n(6), torch.empty(6, 8, device=DEV), g.n(8), g.n(8), torch.zeros(2, device=DEV))
    with pytest.raises(RuntimeError, match="-2"):
        H.short_conv_bwd(v["dy"], v["u"], g.n(8, 4), None, y, g.n(8, 4), None, torch.zeros(2, device=DEV))
    with pytest.raises(ValueError):
        H.short_conv_ws(5, 2, 8, 5, DEV)
    with pytest.raises(ValueError):
        H.layer_norm_ws(5, 20000, DEV)


def test_an_output_beside_an_input_of_the_same_rows_and_one_that_overlaps_it():
    g = Gen(5)
    T, B, D, W = 9, 3, 24, 4
    w, buf = g.n(D, W), g.n(T, B, 2 * D)
    x, ref = buf[..., :D].clone(), torch.empty(T, B, D, device=DEV)
    H.short_conv_fwd(x, w, None, ref)
    with pytest.raises(ValueError, match="shares"):
        H.short_conv_fwd(buf[..., :D], w, None, buf[..., D - 1:2 * D - 1])
    H.short_conv_fwd(buf[..., :D], w, None, buf[..., D:])
    assert torch.equal(buf[..., D:], ref) and torch.equal(buf[..., :D], x)
    rows = g.n(2 * T, D)
    ref = torch.empty(T, D, device=DEV)
    H.layer_norm_fwd(rows[::2], w[:, 0].contiguous(), None, ref)
    with pytest.raises(ValueError, match="shares"):
        H.layer_norm_fwd(rows[:T], w[:, 0].contiguous(), None, rows[T - 1:2 * T - 1])
    H.layer_norm_fwd(rows[::2], w[:, 0].contiguous(), None, rows[1::2])
    assert torch.equal(rows[1::2], ref)
