"""Batched decoding: several sequences a step through one Qwen3-MoE model,
over a paged KV cache of 16- or 32-bit rows, with sampling on the device and,
under a row budget, eviction by accumulated attention weight.

    python -m styx_b200.serve MODEL.gguf --prompt 1,2,3 --prompt 7,8 -n 32
           [--temperature 0.7 --top-k 40 --top-p 0.95 --min-p 0.05 --seed 1]
           [--cache f16] [--experts auto] [--page 64] [--ctx 4096] [--budget 1024 --recent 128 --sinks 4]
           [--chunk 512] [--rope-scaling yarn --rope-factor 4 --rope-orig-ctx 32768]

The defaults hold fewer bits than the f32 of styx_b200.generate, for speed:
K and V as f16 (half the bytes of the cache), and, where the experts' formats
allow, their activations as f16 (grouped tensor-core GEMMs, each expert's
weights read once a step).  --cache f32 --experts f32 undoes both: greedy
tokens are then those of the single-sequence step.

With --chunk the prompts go through the model so many tokens at a time, of as
many sequences as there are (styx_paged_plan hands out rows and pages,
styx_paged_attend_chunk lets every token see its own sequence up to itself),
without it a token of every sequence at a time.

Per token of a step: the embedding rows, then per layer RMSNorm, q / k / v,
styx_paged_append (norms, RoPE, the new row into its page), styx_paged_attend
(with a budget it also accumulates every row's weight), o and the MoE block,
then the output norm, the LM head and styx_sample.  Where a sequence passes
its budget by a page, styx_paged_evict brings every layer down to it and the
freed pages go back to the pool.  The reference decodes one token of one
sequence at a time (crates/model/examples/generate_moe.rs:46-66); its own
step is styx_b200.decode.
"""
from __future__ import annotations

import argparse
import sys
import time
from typing import Optional

import torch

from . import _lib, ops
from .decode import DecodeParams

CACHE_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


class BatchDecoder:
    """n_seqs sequences of one model (the layers of a DecodeModel).  The cache
    holds n_ctx rows per sequence at most; with a budget a sequence is brought
    down to `budget` rows per kv head whenever it has passed it by a page, the
    last n_recent positions and the first n_sink protected.  n_pages: pages of
    the pool (None: as many as all sequences can need at once).  moe_batch:
    the experts as grouped tensor-core GEMMs (f16 operands; None: where their
    formats allow), else token by token in f32.  chunk: tokens of prompts per
    pass (0: a token of every sequence at a time, as decoding).  rope: how heads
    are turned (None: NEOX with the model's base)."""

    def __init__(self, hp: DecodeParams, embd: ops.DenseWeight, layers: list, output_norm: torch.Tensor,
                 head: ops.DenseWeight, n_seqs: int, n_ctx: int, page: int = 64, cache: torch.dtype = torch.float16,
                 budget: int = 0, n_recent: int = 128, n_sink: int = 4, n_pages: Optional[int] = None,
                 moe_batch: Optional[bool] = None, device: int = 0, chunk: int = 0, rope: Optional[ops.Rope] = None):
        if chunk < 0 or (chunk and budget):
            raise ValueError(f"chunks of {chunk} tokens" if chunk < 0 else "prompts in chunks keep all rows: no budget with them")
        if not 1 <= n_seqs <= 64:
            raise ValueError(f"{n_seqs} sequences: 1 to 64")
        if budget and n_recent + n_sink > budget:
            raise ValueError(f"{n_recent} recent and {n_sink} first rows do not fit a budget of {budget}")
        self.hp, self.embd, self.layers, self.output_norm, self.head = hp, embd, layers, output_norm, head
        self.n_seqs, self.page, self.budget, self.n_recent, self.n_sink = n_seqs, page, budget, n_recent, n_sink
        rows = min(n_ctx, budget + page) if budget else n_ctx     # a sequence is evicted to the budget at that many
        self.max_pages = -(-rows // page)
        self.n_rows = rows
        self.n_pages = n_seqs * self.max_pages if n_pages is None else n_pages
        dev = self.device = torch.device("cuda", device)
        f32, i32 = torch.float32, torch.int32
        L, H, kvh, hd = hp.n_layers, hp.n_embd, hp.n_kv_heads, hp.head_dim
        self.pool = torch.empty(2, L, self.n_pages, kvh, page, hd, dtype=cache, device=dev)
        self.table = torch.zeros(n_seqs, self.max_pages, dtype=i32, device=dev)
        self.lens = torch.zeros(n_seqs, dtype=i32, device=dev)
        # the lengths that the caches go by: 0 for the sequences that a step leaves out, so that nothing of theirs is
        # read, and no weight of theirs changes
        self.live = torch.zeros(n_seqs, dtype=i32, device=dev)
        self.kv = [ops.PagedKV(self.pool[0, li], self.pool[1, li], self.table, self.live) for li in range(L)]
        for kv in self.kv[1:]:
            kv.share_workspaces(self.kv[0])
        self.pos = torch.zeros(n_seqs, dtype=i32, device=dev)       # the next token's position
        self.tok = torch.zeros(n_seqs, dtype=i32, device=dev)
        # the host's side of the pages
        self.rows = [0] * n_seqs
        self.pages: list[list[int]] = [[] for _ in range(n_seqs)]
        self.free = list(range(self.n_pages - 1, -1, -1))
        if budget:
            shape = (n_seqs, kvh, self.max_pages * page)
            self.acc = [torch.zeros(shape, dtype=f32, device=dev) for _ in range(L + 1)]    # one spare
            self.row_pos = [torch.zeros(shape, dtype=i32, device=dev) for _ in range(L + 1)]
            self.lens_out = torch.zeros_like(self.lens)
        self.n_q, self.n_k = hp.n_heads * hd, kvh * hd
        self.x = torch.empty(n_seqs, H, dtype=f32, device=dev)
        self.xn = torch.empty_like(self.x)
        self.qkv = torch.empty(n_seqs, self.n_q + 2 * self.n_k, dtype=f32, device=dev)
        self.q = torch.zeros(n_seqs, hp.n_heads, hd, dtype=f32, device=dev)
        self.o = torch.empty_like(self.q)
        self.logits = torch.empty(n_seqs, hp.n_vocab, dtype=f32, device=dev)
        formats = {ly.moe.gate.qtype for ly in layers} | {ly.moe.up.qtype for ly in layers} | {ly.moe.down.qtype for ly in layers}
        can = formats <= {_lib.Q4_K, _lib.Q5_K, _lib.Q6_K} and all(ly.moe.gate.qtype == ly.moe.up.qtype for ly in layers)
        self.moe_batch = can if moe_batch is None else moe_batch
        self.dims = ops.Dims(H, hp.n_ff, hp.n_expert, hp.n_expert_used, hp.norm_topk, hp.rms_eps)
        self.ids = torch.zeros(max(n_seqs, L) * ops.IDS_PER_LAYER, dtype=i32, device=dev)
        self.expert_w = torch.zeros(n_seqs * hp.n_expert_used, dtype=f32, device=dev)
        self.blocks: dict[int, ops.MoeBatch] = {}       # by tokens of a step
        self.chunk, self.rope = chunk, rope
        if chunk:
            self.free_dev = torch.zeros(self.n_pages, dtype=i32, device=dev)
            self.plan = ops.PagedPlan(self.table, page, self.free_dev, chunk)
            self.cx = torch.empty(chunk, H, dtype=f32, device=dev)
            self.cxn = torch.empty_like(self.cx)
            self.cqkv = torch.empty(chunk, self.n_q + 2 * self.n_k, dtype=f32, device=dev)
            self.cq = torch.empty(chunk, hp.n_heads, hd, dtype=f32, device=dev)
            self.co = torch.empty_like(self.cq)
            self.cids = torch.zeros(max(min(64, chunk), L) * ops.IDS_PER_LAYER, dtype=i32, device=dev)
            self.cw = torch.zeros(64 * hp.n_expert_used, dtype=f32, device=dev)
        self.block = None if self.moe_batch else ops.MoeBlock(self.dims, device)

    @classmethod
    def of(cls, model, n_seqs: int, n_ctx: int, **kw) -> "BatchDecoder":
        """Over a DecodeModel's weights."""
        return cls(model.hp, model.embd, model.layers, model.output_norm, model.head, n_seqs, n_ctx, **kw)

    def reset(self) -> None:
        self.lens.zero_()
        self.pos.zero_()
        self.q.zero_()
        for b in range(self.n_seqs):
            self._release(b, 0)

    def _release(self, b: int, rows: int) -> None:
        """Sequence b has `rows` rows; its pages past them are free."""
        self.rows[b] = rows
        keep = -(-rows // self.page)
        self.free.extend(reversed(self.pages[b][keep:]))
        del self.pages[b][keep:]

    def _grow(self, n: int) -> None:
        """One row more for the first n sequences, a page where it starts one;
        ValueError, and nothing changed, where one of them has no room."""
        if not 1 <= n <= self.n_seqs:
            raise ValueError(f"a step of {n} sequences: 1 to {self.n_seqs}")
        starts = []                        # sequences whose new row starts a page
        for b in range(n):
            if self.rows[b] == self.n_rows:
                raise ValueError(f"sequence {b}: KV cache full ({self.n_rows} rows)")
            if self.rows[b] == len(self.pages[b]) * self.page:
                if len(starts) == len(self.free):
                    raise ValueError(f"sequence {b}: no page left of {self.n_pages}")
                starts.append(b)
        for b in starts:
            self.pages[b].append(self.free.pop())
            self.table[b, len(self.pages[b]) - 1] = self.pages[b][-1]
        for b in range(n):
            self.rows[b] += 1
        self.lens[:n] += 1

    def step(self, n: Optional[int] = None) -> torch.Tensor:
        """The tokens tok[:n] of the first n sequences at their next
        positions; returns logits f32 [n][n_vocab].  The other sequences stay
        as they are."""
        hp, hd = self.hp, self.hp.head_dim
        n = self.n_seqs if n is None else n
        self._grow(n)
        self.live[:n] = self.lens[:n]
        if n < self.n_seqs:
            self.live[n:] = 0
        x, xn, pos = self.x[:n], self.xn[:n], self.pos[:n]
        qkv = self.qkv[:n]
        q, k, v = (t.unflatten(1, (-1, hd)) for t in qkv.split((self.n_q, self.n_k, self.n_k), dim=1))
        if self.budget:
            seq, newest = torch.arange(n, device=self.device), (self.lens[:n] - 1).long()
        ops.get_rows(self.embd.qtype, self.embd.data, hp.n_vocab, hp.n_embd, self.tok[:n], out=x)
        for li, ly in enumerate(self.layers):
            w = ly.attn
            ops.rms_norm_into(x, w.attn_norm, hp.rms_eps, xn)
            for t in range(n):
                at = 0
                for m, rows in ((w.wq, self.n_q), (w.wk, self.n_k), (w.wv, self.n_k)):
                    ops.mul_mat_vec(m.qtype, m.data, rows, hp.n_embd, xn[t], y=qkv[t, at:at + rows])
                    at += rows
            self._append(li, q, k, v, pos, self.q[:n])
            if self.budget:
                self.row_pos[li][seq, :, newest] = pos[:, None]
            self.kv[li].attend(self.q, out=self.o, acc=self.acc[li] if self.budget else None)
            for t in range(n):
                ops.mul_mat_vec_add(w.wo.qtype, w.wo.data, hp.n_embd, self.n_q, self.o[t].view(-1), x[t])
            if self.moe_batch:
                if n not in self.blocks:
                    self.blocks[n] = ops.MoeBatch(self.dims, n, self.device.index)
                self.blocks[n].forward(x, ly.moe, self.ids, self.expert_w)
            else:
                for t in range(n):
                    self.block.forward(x[t], ly.moe, li, self.ids)
        pos += 1
        ops.rms_norm_into(x, self.output_norm, hp.rms_eps, xn)
        for t in range(n):
            ops.mul_mat_vec(self.head.qtype, self.head.data, hp.n_vocab, hp.n_embd, xn[t], y=self.logits[t])
        if self.budget and any(self.rows[b] == self.n_rows and self.n_rows > self.budget for b in range(n)):
            self.evict()
        return self.logits[:n]

    def _append(self, li: int, q, k, v, pos, out, seq=None, row=None) -> None:
        hp, w = self.hp, self.layers[li].attn
        self.kv[li].append(q, k, v, pos, None if self.rope else hp.rope_base, w.q_norm if hp.qk_norm else None,
                           w.k_norm if hp.qk_norm else None, hp.rms_eps, seq=seq, row=row, out=out, rope=self.rope)

    def prefill(self, prompts: list) -> torch.Tensor:
        """prompts[b] after what sequence b holds, `chunk` tokens of them all
        at a time; returns the logits f32 [n_seqs][n_vocab] of every sequence's
        last token (of an empty prompt: what the buffer held).  ValueError, and
        nothing changed, where rows or pages do not suffice."""
        hp, hd, dev, page = self.hp, self.hp.head_dim, self.device, self.page
        if not self.chunk:
            raise ValueError("prefill: no chunk size was given")
        if len(prompts) != self.n_seqs:
            raise ValueError(f"{self.n_seqs} prompts expected, got {len(prompts)}")
        left = [len(p) for p in prompts]
        need = 0
        for b, n in enumerate(left):
            if self.rows[b] + n > self.n_rows:
                raise ValueError(f"sequence {b}: KV cache full ({self.n_rows} rows)")
            need += -(-(self.rows[b] + n) // page) - len(self.pages[b])
        if need > len(self.free):
            raise ValueError(f"no page left of {self.n_pages}: {need} needed, {len(self.free)} free")
        plan, i32 = self.plan, torch.int32
        plan.lens.copy_(self.lens)
        plan.next_pos.copy_(self.pos)
        plan.held.copy_(torch.tensor([len(p) for p in self.pages], dtype=i32))
        plan.n_free.fill_(len(self.free))
        self.free_dev[:len(self.free)] = torch.tensor(self.free, dtype=i32)
        want, done = torch.empty(self.n_seqs, dtype=i32, device=dev), [0] * self.n_seqs
        for _ in range(-(-sum(left) // self.chunk)):
            want.copy_(torch.tensor(left, dtype=i32))
            plan.run(want, plan.lens, plan.held, plan.n_free, plan.next_pos)
            # the host follows: the same tokens in the same order, pages from the same end of the stack
            toks, last = [], []
            for b in range(self.n_seqs):
                t = min(left[b], self.chunk - len(toks))
                toks += prompts[b][done[b]:done[b] + t]
                done[b] += t
                left[b] -= t
                self.rows[b] += t
                while len(self.pages[b]) * page < self.rows[b]:
                    self.pages[b].append(self.free.pop())
                if t and not left[b]:
                    last.append((b, len(toks) - 1))
            self.live.copy_(plan.lens)
            T = len(toks)
            x, xn, qkv, o = self.cx[:T], self.cxn[:T], self.cqkv[:T], self.co[:T]
            q, k, v = (t.unflatten(1, (-1, hd)) for t in qkv.split((self.n_q, self.n_k, self.n_k), dim=1))
            ops.get_rows(self.embd.qtype, self.embd.data, hp.n_vocab, hp.n_embd, torch.tensor(toks, dtype=i32, device=dev), out=x)
            for li, ly in enumerate(self.layers):
                w = ly.attn
                ops.rms_norm_into(x, w.attn_norm, hp.rms_eps, xn)
                for t in range(T):
                    at = 0
                    for m, rows in ((w.wq, self.n_q), (w.wk, self.n_k), (w.wv, self.n_k)):
                        ops.mul_mat_vec(m.qtype, m.data, rows, hp.n_embd, xn[t], y=qkv[t, at:at + rows])
                        at += rows
                self._append(li, q, k, v, plan.pos[:T], self.cq[:T], plan.seq[:T], plan.row[:T])
                self.kv[li].attend_chunk(self.cq[:T], plan.start, out=o)
                for t in range(T):
                    ops.mul_mat_vec_add(w.wo.qtype, w.wo.data, hp.n_embd, self.n_q, o[t].view(-1), x[t])
                for t in range(0, T, 64 if self.moe_batch else 1):
                    if self.moe_batch:
                        n = min(64, T - t)
                        if n not in self.blocks:
                            self.blocks[n] = ops.MoeBatch(self.dims, n, dev.index)
                        self.blocks[n].forward(x[t:t + n], ly.moe, self.cids, self.cw)
                    else:
                        self.block.forward(x[t], ly.moe, li, self.cids)
            for b, t in last:
                self.x[b] = x[t]
        self.lens.copy_(plan.lens)
        self.pos.copy_(plan.next_pos)
        ops.rms_norm_into(self.x, self.output_norm, hp.rms_eps, self.xn)
        for b in range(self.n_seqs):
            if prompts[b]:
                ops.mul_mat_vec(self.head.qtype, self.head.data, hp.n_vocab, hp.n_embd, self.xn[b], y=self.logits[b])
        return self.logits

    def evict(self) -> None:
        """Every sequence down to the budget, in every layer."""
        self.live.copy_(self.lens)
        for li, kv in enumerate(self.kv):
            acc, row_pos = self.acc[li], self.row_pos[li]
            kv.evict(acc, row_pos, self.pos, self.budget, self.n_recent, self.n_sink, acc_out=self.acc[-1],
                     pos_out=self.row_pos[-1], lens_out=self.lens_out)
            self.acc[li], self.acc[-1] = self.acc[-1], acc
            self.row_pos[li], self.row_pos[-1] = self.row_pos[-1], row_pos
        self.lens.copy_(self.lens_out)
        for b in range(self.n_seqs):
            self._release(b, min(self.rows[b], self.budget))

    def generate(self, prompts: list, n_predict: int, temperature: float = 0.0, top_k: int = 0, top_p: float = 1.0,
                 min_p: float = 0.0, seed: int = 0) -> list:
        """n_predict tokens after each prompt (temperature 0: the likeliest).
        Without chunks a shorter prompt joins later, so that all prompts end
        with one step."""
        if len(prompts) != self.n_seqs or not all(prompts) or n_predict < 1:
            raise ValueError(f"{self.n_seqs} prompts of one token or more and n_predict > 0 expected")
        self.reset()
        n, dev = self.n_seqs, self.device
        order = sorted(range(n), key=lambda b: -len(prompts[b]))
        longest = len(prompts[order[0]])
        gen = torch.Generator(device=dev).manual_seed(seed)
        full = lambda v, t: torch.full((n,), v, dtype=t, device=dev)   # noqa: E731
        f32 = torch.float32
        settings = (full(temperature, f32), full(top_k, torch.int32), full(top_p, f32), full(min_p, f32))
        logprob = torch.empty(n, dtype=f32, device=dev)
        ids = torch.tensor([[0] * (longest - len(prompts[b])) + list(prompts[b]) for b in order], dtype=torch.int32,
                           device=dev).t().contiguous()
        if self.chunk:
            logits = self.prefill([list(prompts[b]) for b in order])
        else:
            for i in range(longest):
                self.tok.copy_(ids[i])
                logits = self.step(sum(len(prompts[b]) >= longest - i for b in order))
        out = torch.empty(n_predict, n, dtype=torch.int32, device=dev)
        for i in range(n_predict):
            if i:
                logits = self.step()
            ops.sample(logits, torch.rand(n, generator=gen, device=dev), *settings, token=self.tok, logprob=logprob)
            out[i] = self.tok
        self.kv[0].ctx.check_device_error()
        cols = out.t().tolist()
        return [cols[order.index(b)] for b in range(n)]


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("model")
    ap.add_argument("--prompt", action="append", required=True, help="comma-separated token ids; once per sequence")
    ap.add_argument("-n", "--n-predict", type=int, default=32)
    ap.add_argument("--ctx", type=int, default=4096, help="rows a sequence's cache may hold")
    ap.add_argument("--page", type=int, default=64, help="rows of a page")
    ap.add_argument("--cache", choices=sorted(CACHE_TYPES), default="f16", help="element type of the cache")
    ap.add_argument("--experts", choices=["auto", "f32"], default="auto",
                    help="auto: f16 operands where the formats allow, else f32; f32: token by token")
    ap.add_argument("--budget", type=int, default=0, help="rows that stay per sequence and kv head (0: all)")
    ap.add_argument("--recent", type=int, default=128, help="of them: the last so many positions")
    ap.add_argument("--sinks", type=int, default=4, help="and the first so many")
    ap.add_argument("--chunk", type=int, default=0, help="tokens of prompts per pass (0: a token of every prompt at a time)")
    ap.add_argument("--rope-scaling", choices=["linear", "yarn"], help="rotary frequencies for contexts beyond the trained one")
    ap.add_argument("--rope-factor", type=float, default=1.0, help="context by this much longer than the trained one")
    ap.add_argument("--rope-orig-ctx", type=int, default=32768, help="the trained context (yarn)")
    ap.add_argument("--temperature", type=float, default=0.0)
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=1.0)
    ap.add_argument("--min-p", type=float, default=0.0)
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--device", type=int, default=0)
    args = ap.parse_args(argv)

    from . import gguf as G
    torch.cuda.set_device(args.device)
    prompts = [[int(t) for t in p.split(",") if t.strip()] for p in args.prompt]
    g = G.Gguf.open(args.model)
    model, keep = G.load_decode_model(g, 1, args.device)
    g.close()
    rope = ops.Rope(model.hp.head_dim, model.hp.rope_base, scaling=args.rope_scaling, factor=args.rope_factor,
                    orig_ctx=args.rope_orig_ctx, device=args.device) if args.rope_scaling else None
    dec = BatchDecoder.of(model, len(prompts), args.ctx, chunk=args.chunk, rope=rope, page=args.page, cache=CACHE_TYPES[args.cache],
                          budget=args.budget, n_recent=args.recent, n_sink=args.sinks,
                          moe_batch=False if args.experts == "f32" else None, device=args.device)
    t0 = time.perf_counter()
    out = dec.generate(prompts, args.n_predict, args.temperature, args.top_k, args.top_p, args.min_p, args.seed)
    t1 = time.perf_counter()
    for toks in out:
        print(",".join(str(t) for t in toks))
    before = -(-sum(len(p) for p in prompts) // args.chunk) if args.chunk else max(len(p) for p in prompts)
    steps = before + args.n_predict - 1
    print(f"{len(prompts)} sequences, {steps} steps, {steps / (t1 - t0):.1f} steps/s", file=sys.stderr)
    del keep
    return 0


if __name__ == "__main__":
    sys.exit(main())
