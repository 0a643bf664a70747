"""Plain 64-bit forms of the sequence-memory operators, for their tests."""
import torch


def rel(x, ref):
    """2-norm of the difference over the 2-norm of ref (absolute where ref is 0)."""
    x, ref = x.double(), ref.double()
    n = float(ref.norm())
    return float((x - ref).norm()) / (n if n else 1.0)


# ------------------------------------------------------------ linear attention

def scan(q, k, v, log_decay, scale, s0):
    """The recurrence for one sequence: [t, heads, d] inputs in 64 bits, s0 [heads, dk, dv] -> o, final state."""
    s = s0.clone()
    lam = torch.exp(log_decay.double())[:, None, None]
    out = []
    for t in range(q.shape[0]):
        s = lam * s + k[t][:, :, None] * v[t][:, None, :]
        out.append(scale * (q[t][:, :, None] * s).sum(1))
    o = torch.stack(out) if out else q.new_zeros(0, q.shape[1], v.shape[2])
    return o, s


def scan_backward(do, q, k, v, log_decay, scale, s0, ds):
    lam = torch.exp(log_decay.double())[:, None, None]
    s, dq = s0.clone(), torch.zeros_like(q)
    for t in range(q.shape[0]):
        s = lam * s + k[t][:, :, None] * v[t][:, None, :]
        dq[t] = scale * (s * do[t][:, None, :]).sum(2)
    dk, dv, g = torch.zeros_like(k), torch.zeros_like(v), ds.clone()
    for t in range(q.shape[0] - 1, -1, -1):
        g = g + scale * q[t][:, :, None] * do[t][:, None, :]
        dk[t] = (g * v[t][:, None, :]).sum(2)
        dv[t] = (g * k[t][:, :, None]).sum(1)
        g = lam * g
    return dq, dk, dv, g


def sequences(x, lens):
    """[1, total, ...] packed by lens, or [batch, tokens, ...] -> one tensor a sequence, in 64 bits."""
    x = x.double()
    if lens is None:
        return list(x)
    return list(x[0].split(lens))


def linattn(q, k, v, log_decay, scale, state, lens=None):
    h, share = q.shape[2], q.shape[2] // k.shape[2]
    os, ends = [], []
    for i, (a, b, c) in enumerate(zip(*(sequences(x, lens) for x in (q, k, v)))):
        s0 = state[i].double() if state is not None else a.new_zeros(h, q.shape[3], v.shape[3])
        o, s = scan(a, b.repeat_interleave(share, 1), c.repeat_interleave(share, 1), log_decay, scale, s0)
        os.append(o)
        ends.append(s)
    o = torch.cat(os)[None] if lens is not None else torch.stack(os)
    return o, torch.stack(ends) if ends else None


def linattn_backward(do, q, k, v, log_decay, scale, state, dstate, lens=None):
    h, hk = q.shape[2], k.shape[2]
    share, got = h // hk, []
    for i, (d, a, b, c) in enumerate(zip(*(sequences(x, lens) for x in (do, q, k, v)))):
        zero = a.new_zeros(h, q.shape[3], v.shape[3])
        s0 = state[i].double() if state is not None else zero
        ds = dstate[i].double() if dstate is not None else zero
        dq, dk, dv, g = scan_backward(d, a, b.repeat_interleave(share, 1), c.repeat_interleave(share, 1), log_decay, scale, s0, ds)
        got.append((dq, dk.view(-1, hk, share, dk.shape[-1]).sum(2), dv.view(-1, hk, share, dv.shape[-1]).sum(2), g))
    join = (lambda x: torch.cat(x)[None]) if lens is not None else torch.stack
    return [join([g[j] for g in got]) for j in range(3)] + [torch.stack([g[3] for g in got])]


# ------------------------------------------------------------- scaled products

def quantized(x, row_block=1):
    """(values, scales) as fp32, by the definition: scale = max(|x|, 2^-64) / 448, values = e4m3(x / scale)."""
    x = x.float()
    r, c = x.shape
    rb, cb = -(-r // row_block), -(-c // 128)
    p = torch.nn.functional.pad(x, (0, cb * 128 - c, 0, rb * row_block - r)).view(rb, row_block, cb, 128)
    s = p.abs().amax(dim=(1, 3)).clamp_min(2.0 ** -64) * (torch.tensor(1.0 / 448.0, dtype=torch.float32, device=x.device))
    v = (p * (1.0 / s)[:, None, :, None]).reshape(rb * row_block, cb * 128)[:r, :c].to(torch.float8_e4m3fn)
    return v, s


def dequantized(v, s, row_block=1):
    r, c = v.shape
    return v.double() * s.double().repeat_interleave(row_block, 0)[:r].repeat_interleave(128, 1)[:, :c]


# ----------------------------------------------------------------- gated norms

def gatednorm(r, h, gate, alpha, w_post, w_pre, eps, act="silu"):
    """y, z in 64 bits (differentiable)."""
    def norm(x):
        return x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    y = r
    if h is not None:
        u = norm(h)
        u = u * w_post if w_post is not None else u
        u = u * alpha if alpha is not None else u
        if gate is not None:
            u = u * (gate * torch.sigmoid(gate) if act == "silu" else torch.sigmoid(gate))
        y = r + u
    z = norm(y)
    return y, z * w_pre if w_pre is not None else z
