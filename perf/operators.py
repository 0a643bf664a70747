"""The sequence-memory operators of libnrn_b200 at the sizes they are used at.

Three operators, which together are one layer of a memory that reads recorded
activity (libnrn_b200.readout):

* linear attention with a decay for each head (libnrn_b200.linattn): a fast
  Hebbian projection S <- exp(g) S + k v^T, read as o = scale * S^T q.
  ``step`` is one token for each sequence, ``forward`` whole sequences,
  ``backward`` the gradients of ``forward``.
* matrix products in 8-bit floating point (e4m3) with a scale for each block
  of 128 (libnrn_b200.scaled): activations have a scale for each row and 128
  columns, weights one for each 128 x 128 block.  ``product`` is y = x W^T with
  x quantised in the call, ``train`` its gradients dx = dy W and dW = dy^T x,
  with dy and x quantised along the axis that each of the two sums over.
* the norms before and after a block with its gate and residual scale
  (libnrn_b200.gatednorm): y = r + alpha * silu(gate) * norm(h) * w_post and
  z = norm(y) * w_pre in one pass, z also in 8 bits, and the gradients.

``run`` computes them from elementary torch operations in 32 bits, or, with
``own`` set, by the calls a user makes.
"""
import math

import torch

own = False

DEV = "cuda"
E4M3_MAX = 448.0
AMAX_MIN = 2.0 ** -64          # a block's largest magnitude, for its scale, is at least this
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# --------------------------------------------------------------------- cases

def listed():
    return [
        # one recorded session read token by token: the smallest call there is
        {"name": "step one session", "op": "step", "batch": 1, "slots": 1, "heads": 16, "kv_heads": 16,
         "dk": 64, "dv": 64, "dtype": "bf16"},
        # many sessions served at once from a cache of states, key and value heads shared by four
        {"name": "step many sessions", "op": "step", "batch": 192, "slots": 256, "heads": 16, "kv_heads": 4,
         "dk": 128, "dv": 128, "dtype": "bf16"},
        # prompts of very different lengths packed one after the other, each with a state to go on from
        {"name": "packed prompts", "op": "forward", "seqs": 9, "tokens": 12289, "heads": 16, "kv_heads": 16,
         "dk": 128, "dv": 128, "dtype": "bf16", "packed": True},
        # one long recording: few heads, so the time axis has to be split
        {"name": "one long recording", "op": "forward", "seqs": 1, "tokens": 65537, "heads": 8, "kv_heads": 8,
         "dk": 64, "dv": 128, "dtype": "bf16", "packed": False},
        # the backward pass of a training step, key and value heads shared by two
        {"name": "train memory", "op": "backward", "seqs": 2, "tokens": 8190, "heads": 16, "kv_heads": 8,
         "dk": 128, "dv": 128, "dtype": "bf16", "packed": False},
        # three sessions' tokens through one projection: the weights are all that is read
        {"name": "product few rows", "op": "product", "m": 3, "n": 4096, "k": 4096, "dtype": "bf16"},
        # odd everywhere: rows, outputs and a last block of 120 columns
        {"name": "product odd sizes", "op": "product", "m": 515, "n": 1001, "k": 1400, "dtype": "fp16"},
        # a prompt through the widest projection
        {"name": "product prompt", "op": "product", "m": 8192, "n": 8192, "k": 4096, "dtype": "bf16"},
        # both gradients of a projection in a training step
        {"name": "train product", "op": "train", "m": 4097, "n": 2048, "k": 4096, "dtype": "bf16"},
        # one token between two blocks
        {"name": "norm one row", "op": "norm", "rows": 1, "d": 2048, "dtype": "bf16", "scaled": False},
        # a prompt between two blocks, the next block's input in 8 bits
        {"name": "norm prompt", "op": "norm", "rows": 16384, "d": 4096, "dtype": "bf16", "scaled": True},
        # the same in a training step, backward
        {"name": "train norm", "op": "norm_train", "rows": 8191, "d": 2560, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "forward", "forward", "backward", "product", "product", "train", "norm", "norm_train"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    if op == "step":
        share = rng.choice([1, 2, 4])
        heads = share * rng.randint(1, 16 // share)
        batch = _log(rng, 1, 192)
        return {"op": op, "batch": batch, "slots": batch + rng.randint(0, 64), "heads": heads,
                "kv_heads": heads // share, "dk": rng.choice([32, 64, 96, 128]), "dv": rng.choice([32, 64, 80, 128]),
                "dtype": dtype}
    if op in ("forward", "backward"):
        share = rng.choice([1, 1, 2, 4])
        heads = share * rng.randint(1, 16 // share)
        packed = rng.random() < 0.5
        tokens = _log(rng, 16, 12288 if packed or op == "backward" else 65536)
        seqs = min(tokens, rng.choice([1, 2, 5, 16]))
        if not packed:
            tokens = max(1, tokens // seqs)
        return {"op": op, "seqs": seqs, "tokens": tokens, "heads": heads, "kv_heads": heads // share,
                "dk": rng.choice([32, 64, 96, 128]), "dv": rng.choice([32, 64, 80, 128]),
                "dtype": rng.choice(["bf16", "bf16", "bf16", "bf16", "fp16", "fp32"]), "packed": packed}
    if op in ("product", "train"):
        top = 8192 if op == "product" else 4096
        return {"op": op, "m": _log(rng, 1, top), "n": _log(rng, 64, top), "k": _log(rng, 64, 4096), "dtype": dtype}
    d = 8 * _log(rng, 8, 1024)
    case = {"op": op, "rows": _log(rng, 1, min(16384, (16384 * 4096) // d)), "d": d, "dtype": dtype}
    if op == "norm":
        case["scaled"] = rng.random() < 0.5
    return case


# -------------------------------------------------------------------- inputs

def _log_decay(heads):
    """Memories of about 8 to 2,000 tokens, one for each head."""
    x = torch.linspace(3.0, 11.0, heads, dtype=torch.float64) if heads > 1 else torch.tensor([6.0], dtype=torch.float64)
    return torch.log1p(-torch.exp2(-x)).to(torch.float32).to(DEV)


def _lengths(case):
    """Lengths of the packed sequences: from one token to about a third of them all."""
    n, total = case["seqs"], case["tokens"]
    w = [(i + 1) ** 2 for i in range(n)]
    got = [max(1, total * x // sum(w)) for x in w]
    got[0] = 1
    got[-1] += total - sum(got)
    return got


def _e4m3_weights(n, k, randn):
    """Weights as a checkpoint holds them: e4m3 values and a scale for each 128 x 128 block."""
    w = randn(n, k) * (0.5 + torch.rand(n, 1, device=DEV, generator=randn.gen)) / math.sqrt(k)
    nb, kb = -(-n // 128), -(-k // 128)
    p = torch.zeros(nb * 128, kb * 128, device=DEV)
    p[:n, :k] = w
    s = p.view(nb, 128, kb, 128).abs().amax(dim=(1, 3)).clamp_min(AMAX_MIN) / E4M3_MAX
    q = (p.view(nb, 128, kb, 128) / s[:, None, :, None]).reshape(nb * 128, kb * 128)[:n, :k]
    pitch = -(-k // 16) * 16
    values = torch.zeros(n, pitch, device=DEV, dtype=torch.uint8)
    values[:, :k] = q.to(torch.float8_e4m3fn).view(torch.uint8)
    return values.view(torch.float8_e4m3fn)[:, :k], s


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)
    randn.gen = gen

    def cast(x, f=1.0):
        return (x * f).to(dt)

    op = case["op"]
    st = {"op": op, "case": dict(case)}
    if op == "step":
        b, h, hk, dk, dv = case["batch"], case["heads"], case["kv_heads"], case["dk"], case["dv"]
        st["q"], st["k"], st["v"] = cast(randn(b, h, dk)), cast(randn(b, hk, dk)), cast(randn(b, hk, dv))
        st["decay"], st["scale"] = _log_decay(h), dk ** -0.5
        # a sequence that has run for a while; each pass goes on from where the last one left the states
        st["state"] = 4.0 * randn(case["slots"], h, dk, dv)
        st["slots"] = torch.randperm(case["slots"], device=DEV, generator=gen)[:b].to(torch.int32)
    elif op in ("forward", "backward"):
        s, h, hk, dk, dv = case["seqs"], case["heads"], case["kv_heads"], case["dk"], case["dv"]
        shape = (1, case["tokens"]) if case["packed"] else (s, case["tokens"])
        st["q"], st["k"], st["v"] = cast(randn(*shape, h, dk)), cast(randn(*shape, hk, dk)), cast(randn(*shape, hk, dv))
        st["decay"], st["scale"] = _log_decay(h), dk ** -0.5
        st["state"] = 4.0 * randn(s, h, dk, dv)
        lens = _lengths(case) if case["packed"] else [case["tokens"]] * s
        st["lens"] = torch.tensor(lens, device=DEV, dtype=torch.int32)
        st["longest"] = max(lens)
        st["cu"] = None
        if case["packed"]:
            st["cu"] = torch.zeros(s + 1, device=DEV, dtype=torch.int32)
            st["cu"][1:] = st["lens"].cumsum(0)
        if op == "backward":
            st["do"] = cast(randn(*shape, h, dv))
            st["dstate"] = randn(s, h, dk, dv)
    elif op in ("product", "train"):
        m, n, k = case["m"], case["n"], case["k"]
        x = randn(m, k)
        # a few columns that are always large, as activations have them
        x[:, torch.rand(k, device=DEV, generator=gen) < 0.01] *= 20.0
        st["x"] = cast(x)
        st["w"], st["ws"] = _e4m3_weights(n, k, randn)
        if op == "train":
            st["dy"] = cast(randn(m, n), 1e-3)
    else:
        r, d = case["rows"], case["d"]
        st["r"], st["h"], st["gate"] = cast(randn(r, d)), cast(randn(r, d), 3.0), cast(randn(r, d))
        st["alpha"] = 0.3 + 0.1 * randn(d)
        st["w_post"], st["w_pre"] = 1.0 + 0.1 * randn(d), 1.0 + 0.1 * randn(d)
        if op == "norm_train":
            st["dy"], st["dz"] = cast(randn(r, d)), cast(randn(r, d))
    return st


# ---------------------------------------------------------------- plain form

def _powers(decay, n):
    """exp(decay * n), [heads, *n.shape]; n is a tensor of whole numbers."""
    return torch.exp(decay.view(-1, *([1] * n.dim())) * n)


def _heads(x, h):
    """[.., kv heads, d] in 32 bits with each head repeated for the heads that share it."""
    return x.float().repeat_interleave(h // x.shape[-2], dim=-2)


def _scan(q, k, v, decay, scale, s0, off, keep, lens):
    """o_i = scale * (exp(g (i + off)) S0^T q_i + sum_{j <= i} exp(g (i - j)) (q_i . k_j) v_j) for [s, t, heads, d] inputs in
    32 bits, zero from each sequence's length on (``keep``), and the state after its last token; chunks of 64 tokens."""
    s, t, h, dk = q.shape
    dv, c = v.shape[-1], 64
    n = -(-t // c)

    def chunks(x):
        return torch.nn.functional.pad(x, (0, 0, 0, 0, 0, n * c - t)).view(s, n, c, h, -1).permute(0, 3, 1, 2, 4)

    q, k, v = chunks(q * keep), chunks(k * keep), chunks(v * keep)               # [s, h, n, c, d]
    i = torch.arange(c, device=q.device)
    lag = i[:, None] - i[None, :]
    inside = torch.where(lag >= 0, _powers(decay, lag.clamp_min(0)), 0.0)        # [h, c, c]
    to_end = _powers(decay, c - off - i)                                         # [h, c]
    u = (k * to_end[None, :, None, :, None]).transpose(-1, -2) @ v               # [s, h, n, dk, dv]
    a = torch.arange(n, device=q.device)
    gap = a[:, None] - a[None, :] - 1
    between = torch.where(gap >= 0, _powers(decay, gap.clamp_min(0) * c), 0.0)   # [h, n, n]
    x = (between @ u.reshape(s, h, n, dk * dv)).view(s, h, n, dk, dv)
    x = x + _powers(decay, a * c)[None, :, :, None, None] * s0[:, :, None]
    o = ((q @ k.transpose(-1, -2)) * inside[None, :, None]) @ v
    o = scale * (o + _powers(decay, i + off)[None, :, None, :, None] * (q @ x))
    o = o.permute(0, 2, 3, 1, 4).reshape(s, n * c, h, dv)[:, :t]
    left = (lens[:, None] - off - torch.arange(n * c, device=q.device)[None, :]).clamp_min(0)   # [s, n * c]
    w = torch.exp(decay[None, :, None] * left[:, None, :]).view(s, h, n, c, 1)
    end = ((k * w).reshape(s, h, n * c, dk).transpose(-1, -2) @ v.reshape(s, h, n * c, dv))
    end = end + torch.exp(decay[None, :] * lens[:, None])[..., None, None] * s0
    return o, end


def _rows_of(st):
    """Row of the packed arrays for each (sequence, token), whether there is one, and where each sequence's tokens go in reverse."""
    t = torch.arange(st["longest"], device=DEV)
    there = t[None, :] < st["lens"][:, None]
    first = st["cu"][:-1] if st["cu"] is not None else torch.arange(len(st["lens"]), device=DEV) * st["case"]["tokens"]
    return torch.where(there, first[:, None] + t[None, :], 0).long(), there, (st["lens"][:, None] - 1 - t[None, :]).clamp_min(0).long()


def _pad(x, rows):
    return x.reshape(-1, *x.shape[2:])[rows]


def _unpad(x, there, shape):
    return x[there].reshape(*shape[:2], *x.shape[2:])


def _forward_plain(st):
    rows, there, _ = _rows_of(st)
    h, dt = st["q"].shape[2], st["q"].dtype
    keep = there[..., None, None].float()
    q, k, v = (_heads(_pad(st[x], rows), h) for x in "qkv")
    o, end = _scan(q, k, v, st["decay"], st["scale"], st["state"], 1, keep, st["lens"])
    return {"o": _unpad(o, there, st["q"].shape).to(dt), "state": end}


def _backward_plain(st):
    rows, there, back = _rows_of(st)
    h, hk, dt = st["q"].shape[2], st["k"].shape[2], st["q"].dtype
    keep = there[..., None, None].float()
    q, k, v, do = (_heads(_pad(st[x], rows), h) for x in ("q", "k", "v", "do"))

    def flip(x):
        return x.gather(1, back[..., None, None].expand(-1, -1, *x.shape[2:]))

    dq, _ = _scan(do, v, k, st["decay"], st["scale"], st["state"].transpose(-1, -2), 1, keep, st["lens"])
    # the gradients run the other way; what the final state's gradient brings has no factor of the scale
    fq, fk, fv, fdo = flip(q), flip(k), flip(v), flip(do)
    dk, ds = _scan(fv, fdo, fq * st["scale"], st["decay"], 1.0, st["dstate"].transpose(-1, -2), 0, keep, st["lens"])
    dv, _ = _scan(fk, fq * st["scale"], fdo, st["decay"], 1.0, st["dstate"], 0, keep, st["lens"])

    def shared(x):
        x = flip(x)
        return x.view(*x.shape[:2], hk, h // hk, x.shape[-1]).sum(3)

    shape = st["q"].shape
    return {"dq": _unpad(dq, there, shape).to(dt), "dk": _unpad(shared(dk), there, shape).to(dt),
            "dv": _unpad(shared(dv), there, shape).to(dt), "dstate": ds.transpose(-1, -2)}


def _step_plain(st):
    h, at = st["q"].shape[1], st["slots"].long()
    q, k, v = (_heads(st[x], h) for x in "qkv")
    state = st["state"][at] * torch.exp(st["decay"])[None, :, None, None] + k[..., :, None] * v[..., None, :]
    st["state"][at] = state
    o = st["scale"] * (q[..., :, None] * state).sum(-2)
    return {"o": o.to(st["q"].dtype), "state": st["state"]}


def _quantised(x, row_block=1):
    """x in 32 bits as what its e4m3 values and scales stand for: a scale for each ``row_block`` x 128 block."""
    r, c = x.shape
    rp, cp = -(-r // row_block) * row_block, -(-c // 128) * 128
    b = torch.nn.functional.pad(x, (0, cp - c, 0, rp - r)).view(rp // row_block, row_block, cp // 128, 128)
    s = b.abs().amax(dim=(1, 3), keepdim=True).clamp_min(AMAX_MIN) / E4M3_MAX
    v = (b * (1.0 / s)).to(torch.float8_e4m3fn)
    return (v.float() * s).reshape(rp, cp)[:r, :c], v, s


def _weights(st):
    n, k = st["w"].shape
    s = st["ws"].repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return st["w"].float() * s


def _product_plain(st):
    return (_quantised(st["x"].float())[0] @ _weights(st).t()).to(st["x"].dtype)


def _train_plain(st):
    x, dy, dt = st["x"].float(), st["dy"].float(), st["x"].dtype
    dx = _quantised(dy)[0] @ _weights(st)
    dw = _quantised(dy.t())[0] @ _quantised(x.t())[0].t()
    return {"dx": dx.to(dt), "dw": dw.to(dt)}


def _normed(x):
    inv = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    return x * inv, inv


def _norm_plain(st):
    dt = st["r"].dtype
    r, h, gate = st["r"].float(), st["h"].float(), st["gate"].float()
    y = r + st["alpha"] * (gate * torch.sigmoid(gate)) * (_normed(h)[0] * st["w_post"])
    z = _normed(y)[0] * st["w_pre"]
    if not st["case"]["scaled"]:
        return {"y": y.to(dt), "z": z.to(dt)}
    _, v, s = _quantised(z)
    rows, d = z.shape
    return {"y": y.to(dt), "z": v.reshape(rows, -1)[:, :d], "scales": s.view(rows, -1)}


def _norm_train_plain(st):
    dt = st["r"].dtype
    r, h, gate, dy, dz = (st[x].float() for x in ("r", "h", "gate", "dy", "dz"))
    hh, inv_h = _normed(h)
    sig = torch.sigmoid(gate)
    act, u = gate * sig, hh * st["w_post"]
    zh, inv_y = _normed(r + st["alpha"] * act * u)
    dzw = dz * st["w_pre"]
    g = dy + inv_y * (dzw - zh * (dzw * zh).mean(-1, keepdim=True))
    du = g * st["alpha"] * act
    dhh = du * st["w_post"]
    dh = inv_h * (dhh - hh * (dhh * hh).mean(-1, keepdim=True))
    dgate = g * st["alpha"] * u * (sig * (1.0 + gate * (1.0 - sig)))
    return {"dr": g.to(dt), "dh": dh.to(dt), "dgate": dgate.to(dt), "dalpha": (g * act * u).sum(0),
            "dw_post": (du * hh).sum(0), "dw_pre": (dz * zh).sum(0)}


PLAIN = {"step": _step_plain, "forward": _forward_plain, "backward": _backward_plain, "product": _product_plain,
         "train": _train_plain, "norm": _norm_plain, "norm_train": _norm_train_plain}


# ------------------------------------------------------- the framework's calls

def _own(st):
    op = st["op"]
    if op in ("step", "forward", "backward"):
        from libnrn_b200 import linattn
        if op == "step":
            o = linattn.step(st["q"], st["k"], st["v"], st["decay"], st["state"], scale=st["scale"], slots=st["slots"])
            return {"o": o, "state": st["state"]}
        if op == "forward":
            o, end = linattn.forward(st["q"], st["k"], st["v"], st["decay"], scale=st["scale"], state=st["state"],
                                     cu_seqlens=st["cu"])
            return {"o": o, "state": end}
        dq, dk, dv, ds = linattn.backward(st["do"], st["q"], st["k"], st["v"], st["decay"], scale=st["scale"],
                                          state=st["state"], dstate=st["dstate"], cu_seqlens=st["cu"])
        return {"dq": dq, "dk": dk, "dv": dv, "dstate": ds}
    if op in ("product", "train"):
        from libnrn_b200 import scaled
        w = scaled.Scaled(st["w"], st["ws"], row_block=128)
        if op == "product":
            return scaled.product(scaled.quantize(st["x"]), w, dtype=st["x"].dtype)
        dx, dw = scaled.product_backward(st["dy"], st["x"], w, dw_dtype=st["x"].dtype)
        return {"dx": dx, "dw": dw}
    from libnrn_b200 import gatednorm
    kw = {"alpha": st["alpha"], "w_post": st["w_post"], "w_pre": st["w_pre"], "eps": EPS}
    if op == "norm":
        y, z = gatednorm.forward(st["r"], st["h"], st["gate"], scaled=st["case"]["scaled"], **kw)
        return {"y": y, "z": z.values, "scales": z.scales} if st["case"]["scaled"] else {"y": y, "z": z}
    g = gatednorm.backward(st["dy"], st["dz"], st["r"], st["h"], st["gate"], **kw)
    return {"dr": g.residual, "dh": g.h, "dgate": g.gate, "dalpha": g.alpha, "dw_post": g.w_post, "dw_pre": g.w_pre}


def run(state):
    return _own(state) if own else PLAIN[state["op"]](state)


# -------------------------------------------------------------------- 64 bits

def _e4m3(x):
    """x rounded to the nearest e4m3 value (ties to even): 3 fraction bits, exponents from -6."""
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -40))).clamp_min(-6.0)
    step = torch.exp2(e - 3.0)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_quantised(x, row_block=1):
    out, vals = torch.empty_like(x), torch.empty_like(x)
    blocks = -(-x.shape[1] // 128)
    s = torch.empty(x.shape[0], blocks, dtype=x.dtype, device=x.device)
    for b in range(blocks):
        part = x[:, 128 * b:128 * (b + 1)]
        sc = part.abs().amax(1, keepdim=True).clamp_min(AMAX_MIN) / E4M3_MAX
        vals[:, 128 * b:128 * (b + 1)] = _e4m3(part / sc)
        out[:, 128 * b:128 * (b + 1)] = vals[:, 128 * b:128 * (b + 1)] * sc
        s[:, b:b + 1] = sc
    return out, vals, s


def _exact_weights(st):
    n, k = st["w"].shape
    i, j = torch.arange(n, device=DEV) // 128, torch.arange(k, device=DEV) // 128
    return st["w"].double() * st["ws"].double()[i][:, j]


def _exact_memory(st, backward):
    """The recurrence itself, token by token for each sequence."""
    q, k, v = (st[x].double() for x in "qkv")
    h, hk = q.shape[2], k.shape[2]
    lam, sc = torch.exp(st["decay"].double())[:, None, None], st["scale"]
    of = torch.arange(h, device=DEV) // (h // hk)
    flat = {n: x.reshape(-1, *x.shape[2:]) for n, x in (("q", q), ("k", k), ("v", v))}
    lens = st["lens"].tolist()
    firsts = [sum(lens[:i]) for i in range(len(lens))]
    if backward:
        do = st["do"].double().reshape(-1, *st["do"].shape[2:])
        dq, dk, dv = (torch.zeros_like(flat[n]) for n in "qkv")
        ds = torch.empty_like(st["dstate"], dtype=torch.float64)
    else:
        o = torch.zeros(flat["q"].shape[0], h, v.shape[-1], dtype=torch.float64, device=DEV)
        end = torch.empty_like(st["state"], dtype=torch.float64)
    # sequences of one length go together; where none are alike each goes alone
    groups = {}
    for i, n in enumerate(lens):
        groups.setdefault(n, []).append(i)
    for n, ids in groups.items():
        rows = torch.tensor([firsts[i] for i in ids], device=DEV)
        at = torch.tensor(ids, device=DEV)
        s = st["state"].double()[at]
        for t in range(n):
            r = rows + t
            s = torch.addcmul(lam * s, flat["k"][r][:, of, :, None], flat["v"][r][:, of, None, :])
            if backward:
                dq[r] = sc * (s @ do[r][..., None])[..., 0]
            else:
                o[r] = sc * (flat["q"][r][:, :, None, :] @ s)[:, :, 0]
        if not backward:
            end[at] = s
            continue
        g = st["dstate"].double()[at]
        for t in range(n - 1, -1, -1):
            r = rows + t
            g = torch.addcmul(g, sc * flat["q"][r][..., :, None], do[r][..., None, :])
            a = (g @ flat["v"][r][:, of, :, None])[..., 0]
            b = (flat["k"][r][:, of, None, :] @ g)[:, :, 0]
            dk[r] = a.view(len(ids), hk, h // hk, -1).sum(2)
            dv[r] = b.view(len(ids), hk, h // hk, -1).sum(2)
            g = lam * g
        ds[at] = g
    if backward:
        return {"dq": dq.view_as(q), "dk": dk.view_as(k), "dv": dv.view_as(v), "dstate": ds}
    return {"o": o.view(*q.shape[:2], h, -1), "state": end}


def _exact_norm(st):
    f = {x: st[x].double() for x in ("r", "h", "gate", "alpha", "w_post", "w_pre")}
    y = f["r"] + f["alpha"] * f["gate"] / (1.0 + torch.exp(-f["gate"])) * f["h"] / (f["h"].pow(2).mean(1, keepdim=True) + EPS).sqrt() * f["w_post"]
    z = y / (y.pow(2).mean(1, keepdim=True) + EPS).sqrt() * f["w_pre"]
    return f, y, z


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "step":
        h, at = case["heads"], st["slots"].long()
        of = torch.arange(h, device=DEV) // (h // case["kv_heads"])
        state = st["state"].double()
        new = torch.exp(st["decay"].double())[:, None, None] * state[at] + torch.einsum("bhi,bhj->bhij", st["k"].double()[:, of], st["v"].double()[:, of])
        state[at] = new
        return {"o": st["scale"] * torch.einsum("bhi,bhij->bhj", st["q"].double(), new), "state": state}
    if op in ("forward", "backward"):
        lens = _lengths(case) if case["packed"] else [case["tokens"]]
        if sum(lens) * (2 if op == "backward" else 1) > 80000:
            return None
        return _exact_memory(st, op == "backward")
    if op == "product":
        return _exact_quantised(st["x"].double())[0] @ _exact_weights(st).t()
    if op == "train":
        x, dy = st["x"].double(), st["dy"].double()
        return {"dx": _exact_quantised(dy)[0] @ _exact_weights(st),
                "dw": _exact_quantised(dy.t().contiguous())[0] @ _exact_quantised(x.t().contiguous())[0].t()}
    f, y, z = _exact_norm(st)
    if op == "norm":
        if not case["scaled"]:
            return {"y": y, "z": z}
        _, v, s = _exact_quantised(z)
        return {"y": y, "z": v, "scales": s}
    leaf = {n: x.clone().requires_grad_(True) for n, x in f.items()}
    with torch.enable_grad():
        _, y, z = _exact_norm(leaf)
        (y * st["dy"].double()).sum().add((z * st["dz"].double()).sum()).backward()
    names = {"r": "dr", "h": "dh", "gate": "dgate", "alpha": "dalpha", "w_post": "dw_post", "w_pre": "dw_pre"}
    return {names[n]: x.grad for n, x in leaf.items()}


# ----------------------------------------------------------------------- work

def work(case):
    op, e = case["op"], SIZE[case["dtype"]]
    if op == "step":
        b, h, hk, dk, dv = (case[x] for x in ("batch", "heads", "kv_heads", "dk", "dv"))
        return {"bytes": b * (8.0 * h * dk * dv + e * (h * dk + hk * (dk + dv) + h * dv)), "flops": 5.0 * b * h * dk * dv}
    if op in ("forward", "backward"):
        h, hk, dk, dv = (case[x] for x in ("heads", "kv_heads", "dk", "dv"))
        n = case["tokens"] * (1 if case["packed"] else case["seqs"])
        states = 8.0 * case["seqs"] * h * dk * dv
        token = h * (dk + dv) + hk * (dk + dv)
        if op == "forward":      # the recurrence's own products: k v^T into the state, q times the state
            return {"bytes": e * n * token + states, "flops": 4.0 * n * h * dk * dv}
        return {"bytes": e * n * (token + h * dk + hk * (dk + dv)) + 1.5 * states, "flops": 10.0 * n * h * dk * dv}
    if op in ("product", "train"):
        m, n, k = case["m"], case["n"], case["k"]
        w = n * k + 4.0 * -(-n // 128) * -(-k // 128)
        if op == "product":
            return {"bytes": e * (m * k + m * n) + w, "flops": 2.0 * m * n * k}
        return {"bytes": e * (2 * m * k + m * n + n * k) + w, "flops": 4.0 * m * n * k}
    r, d = case["rows"], case["d"]
    if op == "norm":
        out = e * r * d + (r * d + 4.0 * r * -(-d // 128) if case["scaled"] else e * r * d)
        return {"bytes": 3.0 * e * r * d + out + 12.0 * d, "flops": 16.0 * r * d}
    return {"bytes": 8.0 * e * r * d + 24.0 * d, "flops": 40.0 * r * d}
