"""A memory that reads recorded activity: blocks of linear attention with
decay (``linattn``) between gated norms (``gatednorm``), with their projections
in 8 bits (``scaled``), over a network's binned spike counts.

    x_0 = counts W_embed^T                      z_0 = norm(x_0) w_pre_0
    q, k, v, gate = z_i W_in_i^T                o = linattn(q, k, v)
    h = o W_out_i^T
    x_{i+1} = x_i + alpha_i silu(gate) norm(h) w_post_i
    z_{i+1} = norm(x_{i+1}) w_pre_{i+1}         answers = z_last W_head^T

The heads' memories are time constants in seconds, as a neuron's are.  A
``Readout`` reads whole recordings (``read``) or one bin of many sessions at a
time from a cache of states (``step``), and learns by gradients
(``gradients``, ``learn``).

    python -m libnrn_b200.readout        # learns to predict a simulated network's next bin
"""
from __future__ import annotations

import math

import numpy as np
import torch

from . import gatednorm, linattn, scaled
from ._tensors import check_rows, require


def bin_spikes(step: np.ndarray, gid: np.ndarray, n: int, bin_steps: int, bins: int, *, first: int = 0, group: int = 1,
               start: int = 0, device="cuda", dtype=torch.bfloat16) -> torch.Tensor:
    """Spike counts [bins, ceil(n / group)] of neurons first .. first + n - 1 of a raster (``Network.raster``), ``group``
    neighbours together, in ``bins`` bins of ``bin_steps`` steps from step ``start`` on.  bf16, which a ``Readout`` takes,
    holds counts to 256 and rounds larger ones to eight bits; another ``dtype`` for more."""
    width = -(-n // group)
    s = torch.from_numpy(np.ascontiguousarray(step)).to(device).long()
    g = torch.from_numpy(np.ascontiguousarray(gid)).to(device).long() - first
    b = (s - start) // bin_steps
    keep = (g >= 0) & (g < n) & (s >= start) & (b < bins)
    at = b[keep] * width + g[keep] // group
    return torch.bincount(at, minlength=bins * width).view(bins, width).to(dtype)


class Readout:
    """``features`` counts in, ``outputs`` answers out, for each bin of ``bin_s`` seconds.  ``tau``: the shortest and the
    longest memory of the heads, in seconds.  Weights are kept in fp32 and used as e4m3 with block scales."""

    def __init__(self, features: int, outputs: int, *, width: int = 256, heads: int = 4, kv_heads: int | None = None, dk: int = 64,
                 dv: int = 64, blocks: int = 2, bin_s: float = 5e-3, tau=(0.02, 2.0), eps: float = 1e-6, seed: int = 0, device="cuda"):
        kv_heads = heads if kv_heads is None else kv_heads
        require(blocks >= 1 and heads >= 1 and kv_heads >= 1 and heads % kv_heads == 0, "heads must be a multiple of kv_heads")
        require(width % 8 == 0 and dk % 8 == 0 and dv % 8 == 0, "width, dk and dv must be multiples of 8")
        require(0 < tau[0] <= tau[1] and bin_s > 0, "tau: two time constants, the shorter first")
        self.features, self.outputs, self.width, self.eps = features, outputs, width, eps
        self.heads, self.kv_heads, self.dk, self.dv, self.blocks = heads, kv_heads, dk, dv, blocks
        self.parts = (heads * dk, kv_heads * dk, kv_heads * dv, width)          # q, k, v, gate
        self.device = torch.device(device)
        if self.device.index is None:
            self.device = torch.device(self.device.type, torch.cuda.current_device())
        memory = torch.logspace(math.log10(tau[0]), math.log10(tau[1]), heads, dtype=torch.float64)
        self.log_decay = (-bin_s / memory).float().to(self.device)
        gen = torch.Generator(device=self.device).manual_seed(seed)

        def w(n, k, f=1.0):
            return torch.randn(n, k, device=self.device, generator=gen) * (f / math.sqrt(k))

        def ones(f=1.0):
            return torch.full((width,), f, device=self.device)
        self.weights = {"embed": w(width, features), "head": w(outputs, width), "w_pre.%d" % blocks: ones()}
        for i in range(blocks):
            self.weights |= {"in.%d" % i: w(sum(self.parts), width), "out.%d" % i: w(width, heads * dv), "alpha.%d" % i: ones(0.5),
                             "w_pre.%d" % i: ones(), "w_post.%d" % i: ones()}

    def small(self, name: str) -> scaled.Scaled:
        """A projection's weights in 8 bits, as they are now."""
        return scaled.quantize(self.weights[name], row_block=128)

    def quantized(self) -> dict:
        """All projections' weights in 8 bits by name: made once by a caller who reads or steps many times with weights that
        stay, and given to those calls as ``small``.  They do not follow ``weights``."""
        return {n: self.small(n) for n in self.weights if n.split(".")[0] in ("embed", "in", "out", "head")}

    def new_states(self, sessions: int) -> list:
        """Zero states, one tensor [sessions, heads, dk, dv] for each block."""
        return [torch.zeros(sessions, self.heads, self.dk, self.dv, device=self.device) for _ in range(self.blocks)]

    def _split(self, p):
        """q, k, v (views by heads) and the gate of a projection [.., sum(parts)]."""
        q, k, v, gate = p.split(self.parts, dim=-1)
        return (q.unflatten(-1, (self.heads, self.dk)), k.unflatten(-1, (self.kv_heads, self.dk)),
                v.unflatten(-1, (self.kv_heads, self.dv)), gate)

    def _norms(self, i):
        """Parameters of the norms after block i and before the next."""
        w = self.weights
        return {"alpha": w["alpha.%d" % i], "w_post": w["w_post.%d" % i], "w_pre": w["w_pre.%d" % (i + 1)], "eps": self.eps}

    def _through(self, counts, attend, small):
        w = self.small if small is None else small.__getitem__
        x = scaled.product(scaled.quantize(counts), w("embed"))
        _, z = gatednorm.forward(x, w_pre=self.weights["w_pre.0"], eps=self.eps, scaled=True)
        for i in range(self.blocks):
            q, k, v, gate = self._split(scaled.product(z, w("in.%d" % i)))
            o = attend(i, q, k, v)
            h = scaled.product(scaled.quantize(o), w("out.%d" % i))
            x, z = gatednorm.forward(x, h, gate, scaled=True, **self._norms(i))
        return scaled.product(z, w("head"))

    def read(self, counts, states=None, cu_seqlens=None, small=None):
        """(answers [batch, bins, outputs], states) of whole recordings [batch, bins, features] (bf16), or of packed ones
        [1, bins, features] with ``cu_seqlens``, that go on from ``states`` (default: nothing remembered).  ``small``:
        weights in 8 bits that the caller keeps (``quantized``; default: made from ``weights`` in the call)."""
        check_rows(counts, "counts", torch.bfloat16, self.device, (*counts.shape[:2], self.features))
        b, t = counts.shape[:2]
        after = []

        def attend(i, q, k, v):
            o, end = linattn.forward(q.unflatten(0, (b, t)), k.unflatten(0, (b, t)), v.unflatten(0, (b, t)), self.log_decay,
                                     state=None if states is None else states[i], cu_seqlens=cu_seqlens)
            after.append(end)
            return o.reshape(b * t, self.heads * self.dv)
        return self._through(counts.reshape(b * t, self.features), attend, small).view(b, t, self.outputs), after

    def step(self, counts, states, slots=None, small=None):
        """Answers [batch, outputs] for one bin [batch, features] of each session; ``states`` are updated in place
        (session i in ``slots[i]``, default i).  ``small`` as in ``read``."""
        check_rows(counts, "counts", torch.bfloat16, self.device, (counts.shape[0], self.features))
        return self._through(counts, lambda i, q, k, v: linattn.step(q, k, v, self.log_decay, states[i], slots=slots).flatten(1), small)

    def gradients(self, counts, targets, cu_seqlens=None):
        """(loss, gradients by the weights' names) of the mean squared error of ``read``'s answers."""
        check_rows(counts, "counts", torch.bfloat16, self.device, (*counts.shape[:2], self.features))
        b, t = counts.shape[:2]
        require(b * t > 0, "counts: no bins, no mean over them")
        require(targets.numel() == b * t * self.outputs, f"targets: must be {(b, t, self.outputs)}, are {tuple(targets.shape)}")
        c = counts.reshape(b * t, -1)
        w = self.quantized().__getitem__
        x = scaled.product(scaled.quantize(c), w("embed"))
        _, z = gatednorm.forward(x, w_pre=self.weights["w_pre.0"], eps=self.eps)
        kept = []
        for i in range(self.blocks):
            p = scaled.product(scaled.quantize(z), w("in.%d" % i))
            q, k, v, gate = self._split(p)
            qkv = tuple(y.unflatten(0, (b, t)) for y in (q, k, v))
            o, _ = linattn.forward(*qkv, self.log_decay, cu_seqlens=cu_seqlens)
            o = o.reshape(b * t, -1)
            h = scaled.product(scaled.quantize(o), w("out.%d" % i))
            kept.append((x, z, qkv, gate, o, h))
            x, z = gatednorm.forward(x, h, gate, **self._norms(i))
        answers = scaled.product(scaled.quantize(z), w("head"), dtype=torch.float32)
        off = answers - targets.reshape(b * t, -1).float()
        grads = {}
        dz, grads["head"] = scaled.product_backward((off * (2.0 / off.numel())).to(torch.bfloat16), z, w("head"))
        dx = None
        for i in range(self.blocks - 1, -1, -1):
            x, z, qkv, gate, o, h = kept[i]
            g = gatednorm.backward(dx, dz, x, h, gate, **self._norms(i))
            grads["alpha.%d" % i], grads["w_post.%d" % i], grads["w_pre.%d" % (i + 1)] = g.alpha, g.w_post, g.w_pre
            do, grads["out.%d" % i] = scaled.product_backward(g.h, o, w("out.%d" % i))
            dqkv = linattn.backward(do.view(b, t, self.heads, self.dv), *qkv, self.log_decay, cu_seqlens=cu_seqlens)[:3]
            dp = torch.cat([y.reshape(b * t, -1) for y in dqkv] + [g.gate], dim=1)
            dz, grads["in.%d" % i] = scaled.product_backward(dp, z, w("in.%d" % i))
            dx = g.residual
        g = gatednorm.backward(dx, dz, kept[0][0], w_pre=self.weights["w_pre.0"], eps=self.eps)
        grads["w_pre.0"] = g.w_pre
        grads["embed"] = scaled.product_backward(g.residual, c, w("embed"))[1]
        return off.square().mean(), grads

    def learn(self, grads, rate: float) -> None:
        """One step against the gradients, each by its own size: weights move by ``rate`` times their own root mean square."""
        for name, g in grads.items():
            w = self.weights[name]
            w -= rate * w.square().mean().sqrt() * g / g.square().mean().sqrt().clamp_min(1e-30)


def main() -> None:
    from . import workloads
    from .engine import Network
    spec = workloads.brunel(8_000, 2_000, 800, 200)
    bin_steps, bins = 50, 640
    nw = Network.from_spec(spec)
    nw.run(bin_steps * bins)
    step, gid = nw.raster()
    nw.close()
    counts = bin_spikes(step, gid, spec["n_total"], bin_steps, bins, group=50)
    print(f"{len(gid)} spikes of {spec['n_total']} neurons in {bins} bins")
    past, future = counts[None, :-1], counts[None, 1:]
    r = Readout(counts.shape[1], counts.shape[1], bin_s=bin_steps * spec["dt"])
    for k in range(41):
        loss, grads = r.gradients(past, future)
        if k % 10 == 0:
            print(f"step {k}: mean squared error {float(loss):.4f}")
        r.learn(grads, 0.02)
    # one bin at a time gives what the whole recording gives
    whole, _ = r.read(past)
    states, small = r.new_states(1), r.quantized()
    for t in range(past.shape[1]):
        last = r.step(past[:, t], states, small=small)
    scaled.check()
    d = float((last - whole[:, -1]).float().norm() / whole[:, -1].float().norm())
    print(f"last bin read step by step differs by {d:.1e} from the whole recording's")


if __name__ == "__main__":
    main()
