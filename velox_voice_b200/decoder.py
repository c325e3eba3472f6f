"""An autoregressive decoder over encoder frames, on the quantized linears and the paged cache.

What stands behind the CTC head when hypotheses are decoded or rescored token by token (the reference rescores whole
hypotheses with its attention decoder, ``veloxvoice/models/wenet/attention_decoder.py:192-240``): the frames of an utterance are read
once and become a prefix that all of its hypotheses share; each hypothesis then has its own tokens.  A block is

    x += lo(attention(rotate(q), rotate(k), v))     q|k|v of LN(x); keys and values go to pages on the way
    x += w2(swish(w1(LN(x))))

in three uses of the same two operators (:func:`ops.kv_append`, :func:`ops.prefix_attention`): :meth:`HypothesisDecoder.read`
(frames, many rows of a sequence, no prefix), :meth:`~HypothesisDecoder.step` (a token per hypothesis) and
:meth:`~HypothesisDecoder.score` (whole hypotheses at once).

``python -m velox_voice_b200.decoder`` reads an utterance and decodes ten hypotheses of it, with random weights.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Sequence

import torch

from . import ops
from .linear import PackedLinear


@dataclass
class DecoderConfig:
    blocks: int = 6
    d_model: int = 512
    heads: int = 8
    kv_heads: int = 8
    ffn: int = 2048
    vocab: int = 5538
    fmt: str = "mx32"
    page_size: int = 16
    positions: int = 8192  # frames and tokens of a hypothesis together
    eps: float = 1e-5

    @property
    def head_dim(self) -> int:
        return self.d_model // self.heads


def make_weights(cfg: DecoderConfig, seed: int = 0) -> Dict[str, torch.Tensor]:
    """Random weights under the names that the decoder takes, fp32 on the CPU."""
    g = torch.Generator().manual_seed(seed)
    d, w = cfg.d_model, {}

    def linear(name, n, k):
        w[name + ".w"], w[name + ".b"] = 0.04 * torch.randn(n, k, generator=g), 0.02 * torch.randn(n, generator=g)

    def norm(name):
        w[name + ".g"], w[name + ".b"] = 1.0 + 0.05 * torch.randn(d, generator=g), 0.05 * torch.randn(d, generator=g)

    for i in range(cfg.blocks):
        p = f"d{i}."
        linear(p + "qkv", (cfg.heads + 2 * cfg.kv_heads) * cfg.head_dim, d)
        linear(p + "lo", d, d)
        linear(p + "w1", cfg.ffn, d)
        linear(p + "w2", d, cfg.ffn)
        norm(p + "ln1")
        norm(p + "ln2")
    norm("after")
    linear("head", cfg.vocab, d)
    w["embed"] = torch.randn(cfg.vocab, d, generator=g)
    return w


@dataclass
class Utterances:
    """Frames that have been read: their pages (int32 [utterances, pages]) and numbers (int32 [utterances]; `counts` on the host)."""

    table: torch.Tensor
    lengths: torch.Tensor
    pages: List[int]
    counts: List[int]
    released: bool = False


@dataclass
class Hypotheses:
    """`beams` hypotheses of every utterance, in the utterances' order.  `tokens`: how many each has been given, finished or not, counted on the
    host against `max_tokens` (a program that moves `lengths` back moves `tokens` too)."""

    utterances: Utterances
    beams: int
    table: torch.Tensor    # int32 [utterances * beams, pages]
    lengths: torch.Tensor  # int32: tokens in the cache; negative: finished
    starts: torch.Tensor   # int32: position of the first token
    pages: List[int]
    max_tokens: int
    tokens: List[int]
    released: bool = False


class HypothesisDecoder:
    """Weights quantized once, a pool of pages for keys and values of every block."""

    def __init__(self, cfg: DecoderConfig, weights: Dict[str, torch.Tensor], pages: int, device="cuda"):
        self.cfg = cfg
        dev = torch.device(device)

        def pack(name):
            return PackedLinear(weights[name + ".w"].to(dev), weights[name + ".b"].to(dev), cfg.fmt)

        def norm(name):
            return weights[name + ".g"].float().to(dev), weights[name + ".b"].float().to(dev)

        self.blocks = [{**{n: pack(f"d{i}.{n}") for n in ("qkv", "lo", "w1", "w2")}, **{n: norm(f"d{i}.{n}") for n in ("ln1", "ln2")}}
                       for i in range(cfg.blocks)]
        self.after, self.head = norm("after"), pack("head")
        self.embed = weights["embed"].to(dev).bfloat16()
        self.rotary = ops.rotary_table(cfg.positions, cfg.head_dim, device=dev)
        shape = (cfg.blocks, pages, cfg.page_size, cfg.kv_heads, cfg.head_dim)
        self.k_pages = torch.empty(shape, dtype=torch.bfloat16, device=dev)
        self.v_pages = torch.empty(shape, dtype=torch.bfloat16, device=dev)
        self._free = list(range(pages))

    # ---- pages
    def _take(self, tokens: Sequence[int]):
        """Pages for owners of so many tokens each: (table, the ids)."""
        counts = [-(-t // self.cfg.page_size) for t in tokens]
        if sum(counts) > len(self._free):
            raise RuntimeError(f"{sum(counts)} pages wanted, {len(self._free)} of {self.k_pages.shape[1]} are free")
        rows, ids = [], []
        for c in counts:
            mine = [self._free.pop() for _ in range(c)]
            ids += mine
            rows.append(mine + [-1] * (max(counts) - c))
        return torch.tensor(rows, dtype=torch.int32).to(self.k_pages.device), ids

    def release(self, owner) -> None:
        """Hands the pages of utterances or hypotheses back."""
        self._free += owner.pages
        owner.pages, owner.released = [], True

    # ---- the blocks
    def _blocks(self, x: torch.Tensor, table, lengths, *, starts=None, row_offsets=None, prefix_table=None, prefix_lengths=None) -> torch.Tensor:
        """Rows x bf16 [rows, d_model] through all blocks; their keys and values stay in the cache."""
        c = self.cfg
        h, kv, dk = c.heads, c.kv_heads, c.head_dim
        for i, b in enumerate(self.blocks):
            qkv = b["qkv"](ops.ln_quantize(x, *b["ln1"], c.eps, c.fmt)).view(x.shape[0], h + 2 * kv, dk)
            k_pages, v_pages = self.k_pages[i], self.v_pages[i]
            q = ops.kv_append(qkv[:, h:h + kv], qkv[:, h + kv:], k_pages, v_pages, table, lengths, q=qkv[:, :h], rotary=self.rotary,
                              row_offsets=row_offsets, starts=starts)
            ctx = ops.prefix_attention(q, k_pages, v_pages, table, lengths, prefix_table, prefix_lengths, row_offsets=row_offsets)
            x = b["lo"](ops.quantize(ctx.view(x.shape[0], h * dk), c.fmt), residual=x)
            up = b["w1"](ops.ln_quantize(x, *b["ln2"], c.eps, c.fmt), act="swish", out_fmt=c.fmt)
            x = b["w2"](up, residual=x)
        return x

    def read(self, frames: torch.Tensor, counts: Sequence[int]) -> Utterances:
        """Encoder frames bf16 [sum(counts), d_model], one utterance after another, into the cache."""
        if frames.dim() != 2 or frames.shape != (sum(counts), self.cfg.d_model) or min(counts) < 1:
            raise ValueError(f"frames must be [{sum(counts)}, {self.cfg.d_model}] with at least one frame per utterance, got {tuple(frames.shape)}")
        if max(counts) > self.cfg.positions:  # (rows at positions that the table does not have are not stored)
            raise ValueError(f"{max(counts)} frames, but the decoder has {self.cfg.positions} positions")
        dev = self.k_pages.device
        table, ids = self._take(counts)
        try:
            n = torch.tensor(counts, dtype=torch.int32).to(dev)
            offsets = torch.zeros(len(counts) + 1, dtype=torch.int32, device=dev)
            offsets[1:] = n.cumsum(0)
            self._blocks(frames, table, torch.zeros_like(n), row_offsets=offsets)
        except BaseException:
            self._free += ids
            raise
        return Utterances(table, n, ids, list(counts))

    def begin(self, utterances: Utterances, beams: int, max_tokens: int) -> Hypotheses:
        """Room for `beams` hypotheses of every utterance, `max_tokens` each."""
        if beams < 1 or max_tokens < 0:
            raise ValueError(f"beams must be 1 or more and max_tokens 0 or more, got {beams} and {max_tokens}")
        self._held(utterances)
        if max(utterances.counts) + max_tokens > self.cfg.positions:
            raise ValueError(f"{max(utterances.counts)} frames and {max_tokens} tokens, but the decoder has {self.cfg.positions} positions")
        total = beams * utterances.lengths.shape[0]
        table, ids = self._take([max_tokens] * total)
        starts = utterances.lengths.repeat_interleave(beams)
        return Hypotheses(utterances, beams, table, torch.zeros_like(starts), starts, ids, max_tokens, [0] * total)

    @staticmethod
    def _held(*owners) -> None:
        if any(o.released for o in owners):
            raise RuntimeError("the pages have been handed back: they may be another owner's")

    def _grown(self, hyp: Hypotheses, counts: Sequence[int]) -> List[int]:
        """Tokens of every hypothesis with so many more: a token without a place in a page would not be stored."""
        self._held(hyp, hyp.utterances)
        tokens = [t + c for t, c in zip(hyp.tokens, counts)]
        if max(tokens) > hyp.max_tokens:
            raise RuntimeError(f"no room: hypotheses of {hyp.max_tokens} tokens at most, {max(tokens)} wanted")
        return tokens

    def _hidden(self, hyp: Hypotheses, ids: torch.Tensor, row_offsets=None) -> torch.Tensor:
        u = hyp.utterances
        return self._blocks(self.embed[ids], hyp.table, hyp.lengths, starts=hyp.starts, row_offsets=row_offsets, prefix_table=u.table,
                            prefix_lengths=u.lengths)

    def step(self, hyp: Hypotheses, ids: torch.Tensor) -> torch.Tensor:
        """One token per hypothesis (ids [utterances * beams]) -> the likeliest next ones, int32."""
        tokens = self._grown(hyp, [1] * len(hyp.tokens))
        out = self._step(hyp, ids)
        hyp.tokens = tokens
        return out

    def _step(self, hyp: Hypotheses, ids: torch.Tensor) -> torch.Tensor:
        x = self._hidden(hyp, ids)
        hyp.lengths.add_((hyp.lengths >= 0).to(torch.int32))
        return self.head.argmax(ops.ln_quantize(x, *self.after, self.cfg.eps, self.cfg.fmt))

    def score(self, hyp: Hypotheses, ids: torch.Tensor, counts: Sequence[int]) -> torch.Tensor:
        """Whole continuations at once: ids [sum(counts)], hypothesis after hypothesis -> bf16 logits [sum(counts), vocab]."""
        counts = list(counts)
        if len(counts) != len(hyp.tokens) or min(counts) < 0 or sum(counts) != ids.numel():
            raise ValueError(f"counts must be those of {len(hyp.tokens)} hypotheses and sum to {ids.numel()} ids, got {counts}")
        tokens = self._grown(hyp, counts)
        n = torch.tensor(counts, dtype=torch.int32).to(hyp.table.device)
        offsets = torch.zeros(n.numel() + 1, dtype=torch.int32, device=n.device)
        offsets[1:] = n.cumsum(0)
        x = self._hidden(hyp, ids, offsets)
        hyp.lengths.add_(torch.where(hyp.lengths >= 0, n, 0))
        hyp.tokens = tokens
        return self.head(ops.ln_quantize(x, *self.after, self.cfg.eps, self.cfg.fmt))

    def compile_step(self, hyp: Hypotheses):
        """``step`` as a CUDA graph: a function of ids (copied in) that returns the graph's own output."""
        self._held(hyp, hyp.utterances)
        ids = torch.zeros(hyp.lengths.shape[0], dtype=torch.int64, device=hyp.table.device)
        kept = hyp.lengths.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self._step(hyp, ids)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = self._step(hyp, ids)
        hyp.lengths.copy_(kept)

        def run(new_ids: torch.Tensor) -> torch.Tensor:
            tokens = self._grown(hyp, [1] * len(hyp.tokens))
            ids.copy_(new_ids)
            graph.replay()
            hyp.tokens = tokens
            return out

        return run


def main() -> None:
    import argparse

    a = argparse.ArgumentParser(description="Read utterances, decode hypotheses of them (random weights).")
    a.add_argument("--frames", type=int, default=375)
    a.add_argument("--utterances", type=int, default=1)
    a.add_argument("--beams", type=int, default=10)
    a.add_argument("--tokens", type=int, default=32)
    o = a.parse_args()
    cfg = DecoderConfig(positions=o.frames + o.tokens)
    ps = cfg.page_size
    dec = HypothesisDecoder(cfg, make_weights(cfg), pages=o.utterances * (-(-o.frames // ps) + o.beams * -(-o.tokens // ps)))
    frames = torch.randn(o.utterances * o.frames, cfg.d_model, device="cuda").bfloat16()
    utt = dec.read(frames, [o.frames] * o.utterances)
    hyp = dec.begin(utt, o.beams, o.tokens)
    step = dec.compile_step(hyp)
    ids = torch.arange(o.utterances * o.beams, device="cuda") % cfg.vocab
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    said = [ids]
    e0.record()
    for _ in range(o.tokens):
        said.append(step(said[-1]).clone())
    e1.record()
    torch.cuda.synchronize()
    print(f"{o.utterances} x {o.beams} hypotheses over {o.frames} frames: {e0.elapsed_time(e1) / o.tokens * 1e3:.0f} us a token; first hypothesis "
          f"{[int(t[0]) for t in said[1:9]]} ...")


if __name__ == "__main__":
    main()
