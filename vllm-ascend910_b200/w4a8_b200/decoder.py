"""A decoder stack that serves from the paged 8-bit cache on the package's own kernels.

Per layer, with no torch operation between:

    qkv, r = linear_prepared_rms_norm(h, norm1, qkv, residual=r)     norm + int8 codes, GEMM
    q      = kv_write(cache, k, v, ..., q=q, cos_sin=rotary)         rotary + quantised page writes
    a      = attention(q, cache, ...)
    h      = linear_prepared(a, o)                                   codes, GEMM
    gu, r  = linear_prepared_rms_norm(h, norm2, gate_up, residual=r)
    h      = linear_prepared(gu, down, act="swiglu")

and ``rms_norm(h, final, residual=r)`` at the end.  ``Pages`` is the host's side of the
cache: which pages a sequence holds and how long it is.  A step's ``Plan`` carries the
page table, lengths and offsets on the device; every kernel reads them there, so a step
captured in a CUDA graph (``Decoder.capture``) serves later steps of the same shape by
copying the new plan into the old one's tensors.

    python -m w4a8_b200.decoder --layers 4 --batch 16 --prompt 512 --steps 16

runs random weights of QwQ-32B's shapes: prompts, then captured single-token steps.
The reference leaves norms, rotary positions, cache and attention to its serving stack.
"""
from __future__ import annotations

import argparse
import dataclasses
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import kvcache, ops
from .ops import PreparedWeight, _check


@dataclasses.dataclass(frozen=True)
class Config:
    """QwQ-32B's shapes unless given."""
    hidden: int = 5120
    q_heads: int = 40
    kv_heads: int = 8
    head_dim: int = 128
    ffn: int = 27648
    group_size: int = 128
    eps: float = 1e-5
    rope_base: float = 1e6
    rope_scaling: Optional[Dict] = None
    page_size: int = 16
    positions: int = 8192

    @property
    def qkv(self) -> int:
        return (self.q_heads + 2 * self.kv_heads) * self.head_dim

    def projections(self) -> Dict[str, Tuple[int, int]]:
        """(N, K) of a layer's four linears."""
        return {"qkv": (self.qkv, self.hidden), "o": (self.hidden, self.q_heads * self.head_dim),
                "gate_up": (2 * self.ffn, self.hidden), "down": (self.hidden, self.ffn)}


@dataclasses.dataclass
class Layer:
    norm1: torch.Tensor
    qkv: PreparedWeight
    o: PreparedWeight
    norm2: torch.Tensor
    gate_up: PreparedWeight
    down: PreparedWeight


@dataclasses.dataclass
class Plan:
    """One step's batch: sequence s brings ``cu[s + 1] - cu[s]`` tokens, its last ones."""
    page_table: torch.Tensor   # int32 [batch, columns]
    kv_lens: torch.Tensor      # int32 [batch], this step's tokens included
    cu: torch.Tensor           # int32 [batch + 1]
    tokens: int
    max_q_len: int

    def copy_(self, other: "Plan") -> None:
        """Takes over another step of the same shape, for a captured step's replay."""
        if (other.tokens, other.max_q_len, other.kv_lens.shape) != (self.tokens, self.max_q_len, self.kv_lens.shape):
            raise RuntimeError("Plan: the captured step has another shape")
        cols = other.page_table.shape[1]
        if cols > self.page_table.shape[1]:
            raise RuntimeError(f"Plan: {cols} pages a sequence, the captured step has room for "
                               f"{self.page_table.shape[1]}")
        self.page_table[:, :cols] = other.page_table
        self.kv_lens.copy_(other.kv_lens)
        self.cu.copy_(other.cu)


class Pages:
    """The pages of one cache geometry: free ones, and those that each sequence holds in order.

    ``positions``: rows of the rotary table, which no sequence may outgrow (past its end the
    kernels would turn every token by the last row's angles)."""

    def __init__(self, pages: int, page_size: int, positions: Optional[int] = None):
        self.page_size, self.positions = page_size, positions
        self._free: List[int] = list(range(pages))[::-1]
        self._held: Dict[int, List[int]] = {}
        self._len: Dict[int, int] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        return self._len[seq]

    def add(self) -> int:
        """A new, empty sequence."""
        self._next += 1
        self._held[self._next], self._len[self._next] = [], 0
        return self._next

    def release(self, seq: int) -> None:
        """Ends a sequence; its pages are free at once (kernels of later steps run after the earlier ones')."""
        self._free.extend(reversed(self._held.pop(seq)))
        del self._len[seq]

    def plan(self, seqs: Sequence[int], counts: Sequence[int], device, columns: int = 0) -> Plan:
        """Lengthens each sequence by its count and lays out the step; nothing changes when pages run out
        or a sequence would outgrow the positions."""
        _check(len(seqs) == len(counts) and len(seqs) > 0, "Pages: a step needs sequences, and a count for each")
        _check(len(set(seqs)) == len(seqs), "Pages: a sequence can be in a step once")
        _check(all(n > 0 for n in counts), "Pages: each sequence of a step brings at least one token")
        S = self.page_size
        longest = max(self._len[s] + n for s, n in zip(seqs, counts))
        if self.positions is not None and longest > self.positions:
            raise RuntimeError(f"Pages: a sequence of {longest} tokens, the rotary table has {self.positions} positions")
        need = [-(-(self._len[s] + n) // S) - len(self._held[s]) for s, n in zip(seqs, counts)]
        if sum(need) > len(self._free):
            raise RuntimeError(f"Pages: {sum(need)} pages needed, {len(self._free)} free")
        cu = [0]
        for s, n, p in zip(seqs, counts, need):
            self._held[s].extend(self._free.pop() for _ in range(p))
            self._len[s] += n
            cu.append(cu[-1] + n)
        wide = max(columns, max(len(self._held[s]) for s in seqs))
        table = [self._held[s] + [-1] * (wide - len(self._held[s])) for s in seqs]
        put = lambda v: torch.tensor(v, dtype=torch.int32).to(device)                       # noqa: E731
        return Plan(put(table), put([self._len[s] for s in seqs]), put(cu), cu[-1], max(counts))


class Decoder:
    """Layers, their caches and a rotary table on one GPU."""

    def __init__(self, cfg: Config, layers: Sequence[Layer], final_norm: torch.Tensor, pages: int, device="cuda"):
        for L in layers:
            for name, (n, k) in cfg.projections().items():
                w = getattr(L, name)
                _check((w.N, w.K) == (n, k), f"Decoder: {name} must be [{n}, {k}]; got [{w.N}, {w.K}]")
        self.cfg, self.layers, self.final_norm = cfg, list(layers), final_norm
        self.caches = [kvcache.KVCache.empty(pages, cfg.kv_heads, cfg.page_size, cfg.head_dim, device) for _ in layers]
        self.cos_sin = kvcache.rotary_table(cfg.head_dim, cfg.positions, cfg.rope_base, cfg.rope_scaling, device)
        self.pages = Pages(pages, cfg.page_size, cfg.positions)

    def step(self, h: torch.Tensor, plan: Plan) -> torch.Tensor:
        """Embedded tokens bf16 [tokens, hidden], in the plan's order -> the stack's normed output."""
        c = self.cfg
        _check(h.dim() == 2 and tuple(h.shape) == (plan.tokens, c.hidden), f"step: h must be [{plan.tokens}, {c.hidden}]")
        T, D, nq, nk = plan.tokens, c.head_dim, c.q_heads * c.head_dim, c.kv_heads * c.head_dim
        batch = (plan.page_table, plan.kv_lens, plan.cu)
        r = None
        for L, cache in zip(self.layers, self.caches):
            if r is None:
                qkv, r = ops.linear_prepared_rms_norm(h, L.norm1, L.qkv, c.eps), h
            else:
                qkv, r = ops.linear_prepared_rms_norm(h, L.norm1, L.qkv, c.eps, residual=r)
            q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split((nq, nk, nk), 1))
            q = kvcache.kv_write(cache, k, v, *batch, q=q, cos_sin=self.cos_sin)
            a = kvcache.attention(q, cache, *batch, plan.max_q_len)
            h = ops.linear_prepared(a.view(T, nq), L.o)
            gu, r = ops.linear_prepared_rms_norm(h, L.norm2, L.gate_up, c.eps, residual=r)
            h = ops.linear_prepared(gu, L.down, act="swiglu")
        if r is None:
            return ops.rms_norm(h, self.final_norm, c.eps)
        return ops.rms_norm(h, self.final_norm, c.eps, residual=r)[0]

    def capture(self, plan: Plan) -> "Captured":
        """A captured step of the plan's shape.  The plan's own step is not run: nothing is written."""
        return Captured(self, plan)


class Captured:
    """``Decoder.step`` as a CUDA graph; calling it with a plan of the captured shape runs that step."""

    def __init__(self, dec: Decoder, plan: Plan):
        # The graph holds addresses only: what it reads and writes outside its own pool stays alive here, the
        # layers as they were captured too.
        self._keep = (dec, [dataclasses.replace(L) for L in dec.layers], list(dec.caches), dec.final_norm, dec.cos_sin)
        self.plan = dataclasses.replace(plan, page_table=plan.page_table.clone(), kv_lens=plan.kv_lens.clone(),
                                        cu=plan.cu.clone())
        self.h = torch.zeros((plan.tokens, dec.cfg.hidden), dtype=torch.bfloat16, device=plan.kv_lens.device)
        # The workspace has to exist before the capture: one step without any page, which writes
        # nothing and attends to nothing.
        self.plan.page_table.fill_(-1)
        side = torch.cuda.Stream(self.h.device)
        side.wait_stream(torch.cuda.current_stream(self.h.device))
        with torch.cuda.stream(side):
            dec.step(self.h, self.plan)
        torch.cuda.current_stream(self.h.device).wait_stream(side)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.out = dec.step(self.h, self.plan)

    def __call__(self, h: torch.Tensor, plan: Plan) -> torch.Tensor:
        """The step's output; the next call overwrites it."""
        # (copy_ would repeat a row for every token and convert types)
        if h.shape != self.h.shape or h.dtype is not self.h.dtype:
            raise RuntimeError(f"the captured step takes bfloat16 [{self.h.shape[0]}, {self.h.shape[1]}]; "
                               f"got {h.dtype} {list(h.shape)}")
        self.h.copy_(h)
        self.plan.copy_(plan)
        self.graph.replay()
        return self.out


def random_layers(cfg: Config, n: int, seed: int = 0, device="cuda") -> Tuple[List[Layer], torch.Tensor]:
    """Layers of random 4-bit weights, scaled so that each linear keeps its input's size, and a final norm."""
    g = torch.Generator(device=device).manual_seed(seed)
    layers = []
    for _ in range(n):
        ws = {}
        for name, (N, K) in cfg.projections().items():
            codes = torch.randint(-8, 8, (N, K), generator=g, device=device, dtype=torch.int8)
            scale = torch.exp(torch.randn(ops.num_groups(K, cfg.group_size), N, generator=g, device=device) * 0.2) / (
                4.6 * K ** 0.5)
            ws[name] = ops.prepare_weights(ops.pack_int4_grouped(codes, cfg.group_size), scale, None, K, cfg.group_size)
        norms = (torch.rand(2, cfg.hidden, generator=g, device=device) + 0.5).bfloat16()
        layers.append(Layer(norm1=norms[0], norm2=norms[1], **ws))
    return layers, torch.ones(cfg.hidden, dtype=torch.bfloat16, device=device)


def _ms(fn, n: int) -> float:
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    a.record()
    for _ in range(n):
        fn()
    b.record()
    b.synchronize()
    return a.elapsed_time(b) / n


def main(argv: Optional[Sequence[str]] = None) -> int:
    ap = argparse.ArgumentParser(prog="python -m w4a8_b200.decoder", description="prompts and decode steps of a random stack")
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--prompt", type=int, default=512)
    ap.add_argument("--steps", type=int, default=16)
    a = ap.parse_args(argv)
    cfg = Config()
    dev = torch.device("cuda", torch.cuda.current_device())
    total = a.prompt + a.steps + 8
    _check(min(a.layers, a.batch, a.prompt, a.steps) > 0 and total <= cfg.positions, "decoder: sizes out of range")
    layers, final = random_layers(cfg, a.layers, device=dev)
    cols = -(-total // cfg.page_size)
    dec = Decoder(cfg, layers, final, a.batch * cols, dev)
    x = torch.randn(a.prompt, cfg.hidden, device=dev).bfloat16()
    seqs = [dec.pages.add() for _ in range(a.batch)]
    plans = [dec.pages.plan([s], [a.prompt], dev) for s in seqs]
    dec.step(x, plans[0])                                   # warm-up: workspace, kernels; written again below
    prompt_ms = _ms(lambda: [dec.step(x, p) for p in plans], 1) / a.batch
    h = torch.randn(a.batch, cfg.hidden, device=dev).bfloat16()
    plan = dec.pages.plan(seqs, [1] * a.batch, dev, cols)
    run = dec.capture(plan)
    for _ in range(3):
        run(h, plan)
        plan = dec.pages.plan(seqs, [1] * a.batch, dev, cols)
    plans = [plan] + [dec.pages.plan(seqs, [1] * a.batch, dev, cols) for _ in range(a.steps - 1)]
    it = iter(plans)
    step_ms = _ms(lambda: run(h, next(it)), a.steps)
    out = run.out.float()
    print(f"{a.layers} layers, {a.batch} sequences: prompt of {a.prompt} tokens {prompt_ms:.3f} ms "
          f"({a.prompt / prompt_ms * 1e3:.0f} tokens/s), decode step {step_ms * 1e3:.0f} us "
          f"({a.batch / step_ms * 1e3:.0f} tokens/s), output rms {out.square().mean().sqrt().item():.3f}")
    return 0 if torch.isfinite(out).all() and ops.workspace_status(dev) == 0 else 1


if __name__ == "__main__":
    raise SystemExit(main())
