"""The operators of a state-space recurrent core, as a program of this framework calls them: cases, inputs, plain forms.

A recurrent Q network trains on stored sequences of 120 steps x 64 rows (40 burn-in + 80) with hidden size 512 and acts on
one step of 64 to 4 096 environments at a time. A core made of layer norm, a short causal convolution and a selective
state-space scan (inner size 1 024 = 2 x 512) needs each of the three over whole sequences with their gradients, and the
last two for single steps. ``run`` computes them with elementary torch operations in 32 bits where ``own`` is false and
calls ``distributed_rl_amd.ops.hip`` where it is true.
"""
import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5


# ---- cases -------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one acting step of 256 environments through the norm in front of the core: the smallest call, pure latency
        dict(name="norm act 256x512", op="norm", T=1, B=256, D=512, type="bf16", train=False),
        # the same norm over a learner batch, forward and backward
        dict(name="norm train 7680x512", op="norm", T=120, B=64, D=512, type="bf16", train=True),
        # a norm over the conv torso's 3136 features of a learner batch, in the type of the master weights
        dict(name="norm train 7680x3136", op="norm", T=120, B=64, D=3136, type="fp32", train=True),
        # the short convolution of one acting step
        dict(name="conv step 4096x1024", op="conv_step", B=4096, D=1024, W=4, type="bf16"),
        # ... of a learner batch whose sequences run over episode ends
        dict(name="conv train 120x64x1024", op="conv", T=120, B=64, D=1024, W=4, type="bf16", train=True, resets=True, ragged=False),
        # ... of a few long padded sequences, at sizes that divide nothing
        dict(name="conv train 1021x9x771", op="conv", T=1021, B=9, D=771, W=3, type="fp32", train=True, resets=True, ragged=True),
        # one acting step of an actor process with 64 environments: latency
        dict(name="ssm step 64x1024", op="ssm_step", B=64, D=1024, N=16, type="bf16"),
        # ... of an actor engine with 4 096: the state is read and written once
        dict(name="ssm step 4096x1024", op="ssm_step", B=4096, D=1024, N=16, type="bf16"),
        # the target network's unroll: no gradient
        dict(name="ssm fwd 120x64x1024", op="ssm", T=120, B=64, D=1024, N=16, type="bf16", train=False, resets=False, ragged=False),
        # the online network's unroll with its backward pass, over episode ends and padding
        dict(name="ssm train 120x64x1024", op="ssm", T=120, B=64, D=1024, N=16, type="bf16", train=True, resets=True, ragged=True),
        # whole long episodes, few rows
        dict(name="ssm train 4096x2x1024", op="ssm", T=4096, B=2, D=1024, N=16, type="fp32", train=True, resets=False, ragged=False),
        # one very long stream with a large state, forward only
        dict(name="ssm fwd 16001x1x520", op="ssm", T=16001, B=1, D=520, N=40, type="bf16", train=False, resets=False, ragged=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "conv", "conv", "conv_step", "ssm", "ssm", "ssm", "ssm_step"])
    typ = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "norm":
        D = _log_int(rng, 16, 4096)
        rows = _log_int(rng, 16, max(16, min(40000, 20_000_000 // D)))
        return dict(op="norm", T=1, B=rows, D=D, type=typ, train=rng.random() < 0.7)
    if kind == "conv":
        D, B = _log_int(rng, 32, 2048), _log_int(rng, 1, 64)
        T = _log_int(rng, 2, max(2, min(8192, 7_000_000 // (D * B))))
        return dict(op="conv", T=T, B=B, D=D, W=rng.choice([2, 3, 4]), type=typ, train=rng.random() < 0.7,
                    resets=rng.random() < 0.5, ragged=rng.random() < 0.5)
    if kind == "conv_step":
        D = _log_int(rng, 32, 2048)
        return dict(op="conv_step", B=_log_int(rng, 1, max(1, min(4096, 4_000_000 // D))), D=D, W=rng.choice([2, 3, 4]), type=typ)
    if kind == "ssm_step":
        D, N = _log_int(rng, 32, 2048), rng.choice([4, 8, 16, 16, 32, rng.randint(1, 64)])
        return dict(op="ssm_step", B=_log_int(rng, 1, max(1, min(4096, 64_000_000 // (D * N)))), D=D, N=N, type=typ)
    D, B = _log_int(rng, 32, 2048), _log_int(rng, 1, 64)
    N = rng.choice([4, 8, 16, 16, 32, rng.randint(1, 64)])
    T = _log_int(rng, 2, max(2, min(8192, 100_000_000 // (D * B * N))))
    return dict(op="ssm", T=T, B=B, D=D, N=N, type=typ, train=rng.random() < 0.7, resets=rng.random() < 0.5, ragged=rng.random() < 0.5)


# ---- inputs ------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    typ = TYPES[case["type"]]
    B, D = case["B"], case["D"]

    def normal(*shape, dtype=torch.float32, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device=DEV) * scale + shift).to(dtype)

    def empty(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device=DEV)

    s = {"case": dict(case)}
    if case["op"] == "norm":
        rows = case["T"] * B
        s.update(x=normal(rows, D, dtype=typ, scale=1.5, shift=0.3), w=normal(D, scale=0.2, shift=1.0), b=normal(D, scale=0.2),
                 y=empty(rows, D, dtype=typ))
        if case["train"]:
            s.update(dy=normal(rows, D, dtype=typ), mean=empty(rows), rstd=empty(rows), dx=empty(rows, D, dtype=typ), dw=empty(D), db=empty(D))
        return s
    if case["op"] == "conv_step":
        W = case["W"]
        s.update(x=normal(B, D, dtype=typ), w=normal(D, W, scale=W ** -0.5), bias=normal(D, scale=0.1), state=normal(B, W - 1, D, dtype=typ),
                 y=empty(B, D, dtype=typ))
        return s
    if case["op"] == "ssm_step" or case["op"] == "ssm":
        N = case["N"]
        # decay rates -1..-N with some spread and step sizes of 0.001 .. 0.1: the usual start of such a core
        step = torch.exp(torch.rand(D, generator=g, device=DEV) * math.log(100.0) + math.log(1e-3))
        s.update(A=-torch.arange(1, N + 1, device=DEV, dtype=torch.float32) * torch.exp(normal(D, N, scale=0.1)),
                 D=normal(D, scale=0.1, shift=1.0), dt_bias=step + torch.log(-torch.expm1(-step)))
    if case["op"] == "ssm_step":
        N = case["N"]
        bc = normal(B, 2 * N, dtype=typ)
        s.update(u=normal(B, D, dtype=typ), dt=normal(B, D, dtype=typ, scale=0.5), Bm=bc[:, :N], Cm=bc[:, N:], z=normal(B, D, dtype=typ),
                 h=normal(B, D, N, scale=0.3), y=empty(B, D, dtype=typ))
        return s
    T = case["T"]
    t = torch.arange(T, device=DEV)
    s["reset"] = (torch.rand(T, B, generator=g, device=DEV) < 1 / 40).to(torch.uint8) if case["resets"] else None
    s["lengths"] = None
    if case["ragged"]:                           # the first row fills the batch, the second is empty where there are enough rows
        n = (torch.rand(B, generator=g, device=DEV) * 0.75 + 0.25).mul(T).ceil().clamp(max=T).to(torch.int32)
        n[0] = T
        n[2:3] = 0
        s["lengths"] = n
    if case["op"] == "conv":
        W = case["W"]
        xz = normal(T, B, 2 * D, dtype=typ)      # the input projection's two halves: the convolution reads the first
        s.update(x=xz[..., :D], w=normal(D, W, scale=W ** -0.5), bias=normal(D, scale=0.1), state_in=normal(B, W - 1, D, dtype=typ),
                 y=empty(T, B, D, dtype=typ), state_out=empty(B, W - 1, D, dtype=typ))
        if case["train"]:
            s.update(dy=normal(T, B, D, dtype=typ), dx=empty(T, B, D, dtype=typ), dw=empty(D, W), db=empty(D), dstate_in=empty(B, W - 1, D, dtype=typ))
        return s
    N = case["N"]
    xz, bc = normal(T, B, 2 * D, dtype=typ), normal(T, B, 2 * N, dtype=typ)
    s.update(u=normal(T, B, D, dtype=typ), dt=normal(T, B, D, dtype=typ, scale=0.5), Bm=bc[..., :N], Cm=bc[..., N:], z=xz[..., D:],
             h0=normal(B, D, N, scale=0.3), hT=empty(B, D, N), y=empty(T, B, D, dtype=typ))
    if case["train"]:
        s.update(dy=normal(T, B, D, dtype=typ), du=empty(T, B, D, dtype=typ), ddt=empty(T, B, D, dtype=typ), dz=empty(T, B, D, dtype=typ),
                 dB=empty(T, B, N, dtype=typ), dC=empty(T, B, N, dtype=typ), dA=empty(D, N), dD=empty(D), ddt_bias=empty(D), dh0=empty(B, D, N))
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    return globals()[("own_" if own else "plain_") + state["case"]["op"]](state)


def own_norm(s):
    from distributed_rl_amd.ops import hip
    if not s["case"]["train"]:
        hip.layer_norm_fwd(s["x"], s["w"], s["b"], s["y"], eps=EPS)
        return {"y": s["y"]}
    if "ws" not in s:
        s["ws"] = hip.layer_norm_ws(s["x"].shape[0], s["x"].shape[1], s["x"].device)
    hip.layer_norm_fwd(s["x"], s["w"], s["b"], s["y"], mean=s["mean"], rstd=s["rstd"], eps=EPS)
    hip.layer_norm_bwd(s["dy"], s["x"], s["w"], s["mean"], s["rstd"], s["dx"], s["dw"], s["db"], s["ws"])
    return {k: s[k] for k in ("y", "dx", "dw", "db")}


def plain_norm(s):
    x, w = s["x"].float(), s["w"]
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    rstd = torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS)
    n = c * rstd
    out = {"y": (n * w + s["b"]).to(s["x"].dtype)}
    if s["case"]["train"]:
        dy = s["dy"].float()
        dn = dy * w
        dx = (dn - dn.mean(-1, keepdim=True) - n * (dn * n).mean(-1, keepdim=True)) * rstd
        out.update(dx=dx.to(s["x"].dtype), dw=(dy * n).sum(0), db=dy.sum(0))
    return out


def own_conv_step(s):
    from distributed_rl_amd.ops import hip
    hip.short_conv_step(s["x"], s["w"], s["bias"], s["state"], s["y"])
    return {"y": s["y"], "state": s["state"]}


def plain_conv_step(s):
    rows = torch.cat([s["state"], s["x"][:, None]], 1)
    pre = (rows.float() * s["w"].t()).sum(1) + s["bias"]
    s["state"].copy_(rows[:, 1:])
    return {"y": (pre * torch.sigmoid(pre)).to(s["x"].dtype), "state": s["state"]}


def own_conv(s):
    from distributed_rl_amd.ops import hip
    hip.short_conv_fwd(s["x"], s["w"], s["bias"], s["y"], state_in=s["state_in"], state_out=s["state_out"], reset=s["reset"], lengths=s["lengths"])
    if not s["case"]["train"]:
        return {"y": s["y"], "state_out": s["state_out"]}
    if "ws" not in s:
        s["ws"] = hip.short_conv_ws(*s["x"].shape, s["w"].shape[1], s["x"].device)
    hip.short_conv_bwd(s["dy"], s["x"], s["w"], s["bias"], s["dx"], s["dw"], s["db"], s["ws"], state_in=s["state_in"],
                       dstate_in=s["dstate_in"], reset=s["reset"], lengths=s["lengths"])
    return {k: s[k] for k in ("y", "state_out", "dx", "dw", "db", "dstate_in")}


def plain_conv(s):
    T, B, D = s["x"].shape
    W, typ = s["case"]["W"], s["x"].dtype
    live = _live(s)[..., None]                                                          # (T, B, 1): steps before a row's end
    episode = s["reset"].int().cumsum(0) if s["reset"] is not None else torch.zeros(T, B, dtype=torch.int32, device=DEV)
    episode = torch.cat([torch.zeros(W - 1, B, dtype=episode.dtype, device=DEV), episode])
    rows = torch.cat([s["state_in"].transpose(0, 1).float(), torch.where(live, s["x"].float(), 0.0)])
    same = [(episode[k:k + T] == episode[W - 1:])[..., None] for k in range(W)]         # the tap is of the step's own episode
    pre = sum(torch.where(same[k], rows[k:k + T], 0.0) * s["w"][:, k] for k in range(W)) + s["bias"]
    sig = torch.sigmoid(pre)
    n = s["lengths"].long() if s["lengths"] is not None else torch.full((B,), T, device=DEV)
    at = n[None, :] + torch.arange(W - 1, device=DEV)[:, None]                          # (W-1, B): the last inputs before a row's end
    col = torch.arange(B, device=DEV)[None, :]
    tail = torch.where((episode[at, col] == episode[n + W - 2, col[0]])[..., None], rows[at, col], 0.0)
    out = {"y": torch.where(live, pre * sig, 0.0).to(typ), "state_out": tail.transpose(0, 1).to(typ)}
    if s["case"]["train"]:
        dpre = torch.where(live, s["dy"].float() * sig * (1.0 + pre * (1.0 - sig)), 0.0)
        pad = [torch.nn.functional.pad(torch.where(same[k], dpre, 0.0) * s["w"][:, k], (0, 0, 0, 0, k, W - 1 - k)) for k in range(W)]
        drows = sum(pad)
        dw = torch.stack([(torch.where(same[k], rows[k:k + T], 0.0) * dpre).sum((0, 1)) for k in range(W)], 1)
        out.update(dx=drows[W - 1:].to(typ), dw=dw, db=dpre.sum((0, 1)), dstate_in=drows[:W - 1].transpose(0, 1).to(typ))
    return out


def own_ssm_step(s):
    from distributed_rl_amd.ops import hip
    hip.ssm_step(s["u"], s["dt"], s["A"], s["Bm"], s["Cm"], s["h"], s["y"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"])
    return {"y": s["y"], "h": s["h"]}


def plain_ssm_step(s):
    u, z = s["u"].float(), s["z"].float()
    step = _softplus(s["dt"].float() + s["dt_bias"])
    h = torch.exp(step[..., None] * s["A"]) * s["h"] + (step * u)[..., None] * s["Bm"].float()[:, None]
    s["h"].copy_(h)
    y = ((h * s["Cm"].float()[:, None]).sum(-1) + s["D"] * u) * z * torch.sigmoid(z)
    return {"y": y.to(s["u"].dtype), "h": s["h"]}


def own_ssm(s):
    from distributed_rl_amd.ops import hip
    T, B, D = s["u"].shape
    N, train = s["case"]["N"], s["case"]["train"]
    if "ws" not in s:
        s["ws"] = hip.ssm_scan_ws(T, B, D, N, s["u"].device, train=train)
        s["ckpt"] = hip.ssm_scan_ckpt(T, B, D, N, s["u"].device) if train else None
    hip.ssm_scan_fwd(s["u"], s["dt"], s["A"], s["Bm"], s["Cm"], s["y"], s["ws"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"], h0=s["h0"],
                     hT=s["hT"], reset=s["reset"], lengths=s["lengths"], ckpt=s["ckpt"])
    if not train:
        return {"y": s["y"], "hT": s["hT"]}
    hip.ssm_scan_bwd(s["dy"], s["u"], s["dt"], s["A"], s["Bm"], s["Cm"], s["ckpt"], s["du"], s["ddt"], s["dA"], s["dB"], s["dC"], s["ws"],
                     D=s["D"], dD=s["dD"], z=s["z"], dz=s["dz"], dt_bias=s["dt_bias"], ddt_bias=s["ddt_bias"], dh0=s["dh0"],
                     reset=s["reset"], lengths=s["lengths"])
    return {k: s[k] for k in ("y", "hT", "du", "ddt", "dz", "dB", "dC", "dA", "dD", "ddt_bias", "dh0")}


def plain_ssm(s):
    typ = s["u"].dtype
    live = _live(s)[..., None]
    u, z, Bm, Cm = (torch.where(live, s[k].float(), 0.0) for k in ("u", "z", "Bm", "Cm"))
    pre = torch.where(live, s["dt"].float(), 0.0) + s["dt_bias"]
    step = torch.where(live, _softplus(pre), 0.0)
    decay = torch.exp(step[..., None] * s["A"])                                         # (T, B, D, N)
    if s["reset"] is not None:
        decay = torch.where((live & (s["reset"] != 0)[..., None])[..., None], 0.0, decay)
    add = (step * u)[..., None] * Bm[:, :, None]
    add[0] += decay[0] * s["h0"]
    h = _scan(decay, add)
    sig = torch.sigmoid(z)
    inner = (h * Cm[:, :, None]).sum(-1) + s["D"] * u
    out = {"y": (inner * z * sig).to(typ), "hT": h[-1]}
    if s["case"]["train"]:
        dy = torch.where(live, s["dy"].float(), 0.0)
        ds = dy * z * sig
        g = _scan(torch.cat([torch.zeros_like(decay[:1]), decay[1:].flip(0)]), (ds[..., None] * Cm[:, :, None]).flip(0)).flip(0)
        carry = g * decay                                                               # dL/dh of the step before
        w = carry * torch.cat([s["h0"][None], h[:-1]])
        dBu = (g * Bm[:, :, None]).sum(-1)
        dstep = (w * s["A"]).sum(-1) + u * dBu
        dpre = torch.where(live, dstep * torch.sigmoid(pre), 0.0)
        out.update(du=(s["D"] * ds + step * dBu).to(typ), ddt=dpre.to(typ), dz=(dy * inner * sig * (1.0 + z * (1.0 - sig))).to(typ),
                   dB=(g * (step * u)[..., None]).sum(2).to(typ), dC=(ds[..., None] * h).sum(2).to(typ),
                   dA=(w * step[..., None]).sum((0, 1)), dD=(ds * u).sum((0, 1)), ddt_bias=dpre.sum((0, 1)), dh0=carry[0])
    return out


def _live(s):
    T, B = s["case"]["T"], s["case"]["B"]
    if s["lengths"] is None:
        return torch.ones(T, B, dtype=torch.bool, device=DEV)
    return torch.arange(T, device=DEV)[:, None] < s["lengths"][None, :]


def _softplus(x):
    return x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))


def _scan(a, b):
    """h[t] = a[t] h[t-1] + b[t] along dim 0 with h[-1] = 0: pairs of steps are joined, and their scan gives every second h."""
    T = a.shape[0]
    if T == 1:
        return b
    n = T // 2 * 2
    h = torch.empty_like(b)
    h[0] = b[0]
    h[1:n:2] = _scan(a[1:n:2] * a[0:n:2], a[1:n:2] * b[0:n:2] + b[1:n:2])
    h[2::2] = a[2::2] * h[1:T - 1:2] + b[2::2]
    return h


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    v = {k: (x.double() if torch.is_tensor(x) and x.is_floating_point() else x) for k, x in s.items()}
    return globals()["exact_" + case["op"]](case, v)


def exact_norm(case, v):
    x = v["x"]
    var, mean = torch.var_mean(x, dim=-1, unbiased=False, keepdim=True)
    sd = (var + EPS).sqrt()
    out = {"y": (x - mean) / sd * v["w"] + v["b"]}
    if case["train"]:
        n, gy = (x - mean) / sd, v["dy"] * v["w"]
        out["dx"] = (gy - gy.sum(-1, keepdim=True) / case["D"] - n * ((gy * n).sum(-1, keepdim=True) / case["D"])) / sd
        out["dw"], out["db"] = torch.einsum("md,md->d", v["dy"], n), v["dy"].sum(0)
    return out


def _ends(case, v):
    return v["lengths"].tolist() if v["lengths"] is not None else [case["T"]] * case["B"]


def exact_conv_step(case, v):
    W = case["W"]
    pre = v["bias"] + v["w"][:, W - 1] * v["x"]
    for k in range(W - 1):
        pre = pre + v["w"][:, k] * v["state"][:, k]
    return {"y": pre / (1 + torch.exp(-pre)), "state": torch.stack([v["state"][:, k] for k in range(1, W - 1)] + [v["x"]], 1)}


def exact_conv(case, v):
    T, B, W = case["T"], case["B"], case["W"]
    hist = [v["state_in"][:, k] for k in range(W - 1)]
    end = torch.tensor(_ends(case, v), device=DEV)
    pres, taps, states = [], [], [torch.stack(hist, 1)]
    for t in range(T):
        if v["reset"] is not None:
            hist = [torch.where((v["reset"][t] != 0)[:, None], 0.0, x) for x in hist]
        row = hist + [v["x"][t]]
        taps.append(row)
        pres.append(v["bias"] + sum(row[k] * v["w"][:, k] for k in range(W)))
        hist = row[1:]
        states.append(torch.stack(hist, 1))
    pre = torch.stack(pres)
    live = (torch.arange(T, device=DEV)[:, None] < end[None, :])[..., None]
    out = {"y": torch.where(live, pre / (1 + torch.exp(-pre)), 0.0),
           "state_out": torch.stack([states[n][b] for b, n in enumerate(end.tolist())])}
    if case["train"]:
        sig = 1 / (1 + torch.exp(-pre))
        dpre = torch.where(live, v["dy"] * (sig + pre * sig * (1 - sig)), 0.0)
        out["dw"] = torch.stack([sum((dpre[t] * taps[t][k]).sum(0) for t in range(T)) for k in range(W)], 1)
        out["db"] = dpre.sum(1).sum(0)
        drow = torch.zeros(T + W - 1, B, case["D"], dtype=torch.float64, device=DEV)
        for k in range(W):
            for t in range(T):
                ok = torch.ones(B, dtype=torch.bool, device=DEV)
                if v["reset"] is not None:                      # the tap is W-1-k steps back: no episode may start in between
                    for r in range(max(0, t - (W - 1 - k) + 1), t + 1):
                        ok &= v["reset"][r] == 0
                drow[t + k] += torch.where(ok[:, None], dpre[t] * v["w"][:, k], 0.0)
        out["dx"], out["dstate_in"] = drow[W - 1:], drow[:W - 1].transpose(0, 1)
    return out


def exact_ssm_step(case, v):
    step = torch.log(1 + torch.exp(v["dt"] + v["dt_bias"]))
    h = v["h"] * torch.exp(step.unsqueeze(2) * v["A"].unsqueeze(0)) + step.unsqueeze(2) * v["u"].unsqueeze(2) * v["Bm"].unsqueeze(1)
    y = torch.einsum("bdn,bn->bd", h, v["Cm"]) + v["u"] * v["D"]
    return {"y": y * v["z"] / (1 + torch.exp(-v["z"])), "h": h}


def exact_ssm(case, v):
    T, B = case["T"], case["B"]
    end = torch.tensor(_ends(case, v), device=DEV)
    h, hs, ys = v["h0"], [], []
    for t in range(T):
        ok = (t < end)[:, None, None]
        step = torch.log(1 + torch.exp(v["dt"][t] + v["dt_bias"]))
        old = h if v["reset"] is None else h * (v["reset"][t] == 0)[:, None, None]
        new = torch.exp(step[..., None] * v["A"]) * old + (step * v["u"][t])[..., None] * v["Bm"][t][:, None]
        h = torch.where(ok, new, h)
        s = (h * v["Cm"][t][:, None]).sum(-1) + v["D"] * v["u"][t]
        ys.append(torch.where(ok[..., 0], s * v["z"][t] / (1 + torch.exp(-v["z"][t])), 0.0))
        if case["train"]:
            hs.append(h)
    out = {"y": torch.stack(ys), "hT": h}
    if not case["train"]:
        return out
    grads = {k: [None] * T for k in ("du", "ddt", "dz", "dB", "dC")}
    dA, dD, dbias, dh = torch.zeros_like(v["A"]), torch.zeros_like(v["D"]), torch.zeros_like(v["D"]), torch.zeros_like(h)
    for t in range(T - 1, -1, -1):
        ok = (t < end)[:, None].to(torch.float64)
        e = torch.exp(v["dt"][t] + v["dt_bias"])
        step, sig = torch.log(1 + e), 1 / (1 + torch.exp(-v["z"][t]))
        keep = ok if v["reset"] is None else ok * (v["reset"][t] == 0)[:, None]
        old = (hs[t - 1] if t else v["h0"]) * keep[..., None]
        dy, u, z = v["dy"][t] * ok, v["u"][t], v["z"][t]
        s = (hs[t] * v["Cm"][t][:, None]).sum(-1) + v["D"] * u
        ds = dy * z * sig
        gh = dh + ds[..., None] * v["Cm"][t][:, None]
        a = torch.exp(step[..., None] * v["A"])
        gh_b = (gh * v["Bm"][t][:, None]).sum(-1)
        dstep = ((gh * a * old * v["A"]).sum(-1) + u * gh_b) * ok
        dpre = dstep * e / (1 + e)
        grads["du"][t], grads["ddt"][t] = v["D"] * ds + step * gh_b * ok, dpre
        grads["dz"][t] = dy * s * sig * (1 + z * (1 - sig))
        grads["dB"][t] = (gh * (step * u * ok)[..., None]).sum(1)
        grads["dC"][t] = (hs[t] * ds[..., None]).sum(1)
        dA += (gh * a * old * (step * ok)[..., None]).sum(0)
        dD += (ds * u).sum(0)
        dbias += dpre.sum(0)
        dh = torch.where(ok[..., None] > 0, gh * a * keep[..., None], dh)
    out.update({k: torch.stack(x) for k, x in grads.items()})
    out.update(dA=dA, dD=dD, ddt_bias=dbias, dh0=dh)
    return out


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    e = 2 if case["type"] == "bf16" else 4
    B, D = case["B"], case["D"]
    if case["op"] == "norm":
        n = case["T"] * B * D
        return {"bytes": n * e * (5 if case["train"] else 2) + D * (16 if case["train"] else 8), "flops": n * (22 if case["train"] else 8)}
    if case["op"] == "conv_step":
        W = case["W"]
        return {"bytes": B * D * e * 2 * W + D * (W + 1) * 4, "flops": B * D * (2 * W + 6)}
    if case["op"] == "ssm_step":
        N = case["N"]
        return {"bytes": B * D * (4 * e + 8 * N) + B * 2 * N * e + D * (N + 2) * 4, "flops": B * D * (7 * N + 20)}
    n = case["T"] * B * D
    live = 0.625 if case["ragged"] else 1.0      # the share of steps before their rows' ends, on average: only those are read and computed
    if case["op"] == "conv":
        W = case["W"]
        state = B * (W - 1) * D * e
        if not case["train"]:
            return {"bytes": n * e * (1 + live) + 2 * state + D * (W + 1) * 4, "flops": n * live * (2 * W + 6)}
        return {"bytes": n * e * (2 + 2 * live) + 3 * state + D * (W + 1) * 8, "flops": n * live * (8 * W + 16)}
    N = case["N"]
    state, bc = B * D * N * 4, case["T"] * B * 2 * N * e
    if not case["train"]:
        return {"bytes": n * e * (1 + 3 * live) + bc * live + 2 * state + D * (N + 2) * 4, "flops": n * live * (7 * N + 20)}
    return {"bytes": n * e * (4 + 4 * live) + bc * (1 + live) + 3 * state + D * (N + 2) * 8, "flops": n * live * (21 * N + 60)}
