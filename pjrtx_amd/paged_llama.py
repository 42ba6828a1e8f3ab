"""Serving many sequences with the llama-like decoder of llama_like.py: a paged
key-value cache and the operator custom calls.

The cache of a layer is two pools of pages [pages, kv_heads, page_size,
head_dim]; a sequence holds any pages, named by its row of the page table, and
is as long as it is: no sequence reserves max_len. Each block is

  (h, x) = add_rms_norm(x, last block's output)     the residual stream is x
  q, k, v = h.wq, h.wk, h.wv; RoPE
  pages = paged_append(pages, k, v, slots)          in place (donated)
  o = paged_attention(q, pages, table, lengths)     (a prompt: within itself)
  (h, x) = add_rms_norm(o.wo, x); the SwiGLU FFN

and the logits go to an argmax and to token_logprobs. Two programs:

* **prefill** of one prompt of up to `chunk` tokens: `(weights..., tokens
  [chunk], targets [chunk], count, table row [1, M], pages...)`; rows at or
  behind `count` are padding and touch no page. `targets` are the tokens to
  score (each prompt token's successor; -1 where there is none).
* **decode** of one token for each of `batch` places: `(weights..., tokens
  [B], positions [B], table [B, M], pages...)`; a negative position is an
  empty place.

Both return `(next tokens, logits, log probabilities of the targets or of the
next tokens, their entropies, the likeliest tokens' log probabilities and ids,
pages...)`.

Key and value heads may be fewer than query heads (`kv_heads`).
"""
from __future__ import annotations

from dataclasses import dataclass

import numpy as np

from .hlo import Builder, T
from .llama_like import LlamaConfig, rope_inv_freq

SDPA = "pjrtx.mlx_metal.scaled_dot_product_attention"


@dataclass(frozen=True)
class PagedConfig:
    model: LlamaConfig = LlamaConfig()
    kv_heads: int = 16
    batch: int = 8
    page_size: int = 16
    pages: int = 512
    chunk: int = 128      # longest prompt
    top_k: int = 5        # likeliest tokens reported

    @property
    def table_width(self) -> int:
        return -(-self.model.max_len // self.page_size)

    @property
    def pool_shape(self) -> tuple[int, ...]:
        return (self.pages, self.kv_heads, self.page_size, self.model.head_dim)


def weight_shapes(cfg: PagedConfig) -> list[tuple[str, tuple[int, ...]]]:
    """llama_like's weights, wk and wv of kv_heads."""
    m = cfg.model
    d, q, kv, f = m.d_model, m.qdim, cfg.kv_heads * m.head_dim, m.ffn
    layer = {"attn_norm": (d,), "wq": (d, q), "wk": (d, kv), "wv": (d, kv), "wo": (q, d), "ffn_norm": (d,),
             "w1": (d, f), "w3": (d, f), "w2": (f, d)}
    out = [("embed", (m.vocab, d))]
    for i in range(m.layers):
        out += [(f"l{i}.{n}", s) for n, s in layer.items()]
    return out + [("final_norm", (d,)), ("lm_head", (d, m.vocab))]


class _Model:
    def __init__(self, b: Builder, cfg: PagedConfig):
        self.b, self.cfg = b, cfg
        self.w = {n: b.param(s, "bf16") for n, s in weight_shapes(cfg)}

    def pools(self) -> list[T]:
        return [self.b.param(self.cfg.pool_shape, "bf16", donate=True) for _ in range(2 * self.cfg.model.layers)]

    def mm(self, x: T, w: T) -> T:
        return self.b.dot_general(x, w, contract=((1,), (0,)))

    def embed(self, tokens: T) -> T:
        b, m = self.b, self.cfg.model
        return b.gather(self.w["embed"], b.reshape(tokens, (tokens.shape[0], 1)), offset_dims=[1],
                        collapsed_slice_dims=[0], start_index_map=[0], index_vector_dim=1, slice_sizes=[1, m.d_model])

    def rope_tables(self, pos: T) -> tuple[T, T]:
        b, m = self.b, self.cfg.model
        n, half = pos.shape[0], m.head_dim // 2
        inv = b.dense(rope_inv_freq(m).tolist(), "f32", (half,))
        ang = b.multiply(b.broadcast_in_dim(b.convert(pos, "f32"), (n, half), [0]),
                         b.broadcast_in_dim(inv, (n, half), [1]))
        c, s = b.cosine(ang), b.sine(ang)
        return b.concatenate([c, c], 1), b.concatenate([s, s], 1)

    def rope(self, x: T, cos: T, sin: T) -> T:
        """x [N, H, D] bf16: x*cos + rotate_half(x)*sin in f32, to bf16."""
        b = self.b
        n, h, d = x.shape
        xf = b.convert(x, "f32")
        x1 = b.slice(xf, [0, 0, 0], [n, h, d // 2])
        x2 = b.slice(xf, [0, 0, d // 2], [n, h, d])
        rot = b.concatenate([b.negate(x2), x1], 2)
        c, s = (b.broadcast_in_dim(t, xf.shape, [0, 2]) for t in (cos, sin))
        return b.convert(b.add(b.multiply(xf, c), b.multiply(rot, s)), "bf16")

    def slots(self, table: T, rows: T, pos: T, live: T) -> T:
        """The pool slot of each position, -1 where it is not live or the table
        names no page."""
        b, cfg = self.b, self.cfg
        n = pos.shape[0]
        at = b.select(live, pos, b.scalar_like(0, pos))
        size = b.scalar_like(cfg.page_size, at)
        idx = b.concatenate([b.reshape(rows, (n, 1)), b.reshape(b.divide(at, size), (n, 1))], 1)
        page = b.gather(table, idx, offset_dims=[], collapsed_slice_dims=[0, 1], start_index_map=[0, 1],
                        index_vector_dim=1, slice_sizes=[1, 1])
        slot = b.add(b.multiply(page, size), b.remainder(at, size))
        held = b.and_(live, b.compare("GE", page, b.scalar_like(0, page)))
        return b.select(held, slot, b.scalar_like(-1, slot))

    def heads(self, x: T, count: int) -> T:
        return self.b.reshape(x, (x.shape[0], count, self.cfg.model.head_dim))

    def blocks(self, tokens: T, pos: T, slots: T, pools: list[T], attend):
        """The decoder's rows after the last block: the final norm's input as
        (output, residual), and the pools. attend(q, k, v, k pool, v pool)."""
        b, cfg, m = self.b, self.cfg, self.cfg.model
        cos, sin = self.rope_tables(pos)
        out, x = None, self.embed(tokens)
        pools = list(pools)
        for i in range(m.layers):
            w = lambda n: self.w[f"l{i}.{n}"]  # noqa: E731
            if out is None:
                (h,) = b.add_rms_norm(x, None, w("attn_norm"), m.eps)
            else:
                h, x = b.add_rms_norm(out, x, w("attn_norm"), m.eps)
            q = self.rope(self.heads(self.mm(h, w("wq")), m.heads), cos, sin)
            k = self.rope(self.heads(self.mm(h, w("wk")), cfg.kv_heads), cos, sin)
            v = self.heads(self.mm(h, w("wv")), cfg.kv_heads)
            pools[2 * i], pools[2 * i + 1] = b.paged_append(pools[2 * i], pools[2 * i + 1], k, v, slots)
            o = attend(q, k, v, pools[2 * i], pools[2 * i + 1])
            h, x = b.add_rms_norm(self.mm(b.reshape(o, (x.shape[0], m.qdim)), w("wo")), x, w("ffn_norm"), m.eps)
            g = b.convert(self.mm(h, w("w1")), "f32")
            act = b.multiply(b.convert(b.multiply(g, b.logistic(g)), "bf16"), self.mm(h, w("w3")))
            out = self.mm(act, w("w2"))
        return out, x, pools

    def answer(self, h: T, targets: T | None):
        """Next tokens, logits and log probabilities of the rows h."""
        b = self.b
        logits = self.mm(h, self.w["lm_head"])
        _, tok = b.argmax(logits, 1, "s32")
        return [tok, logits, *self.scores(logits, tok if targets is None else targets)]

    def scores(self, logits: T, targets: T):
        lp, entropy, _, *top = self.b.token_logprobs(logits, targets, self.cfg.top_k)
        return [lp, entropy, *top]


def decode_program(cfg: PagedConfig) -> str:
    b = Builder("jit_paged_decode")
    m = _Model(b, cfg)
    tokens, pos = b.param((cfg.batch,), "s32"), b.param((cfg.batch,), "s32")
    table = b.param((cfg.batch, cfg.table_width), "s32")
    pools = m.pools()
    live = b.compare("GE", pos, b.scalar_like(0, pos))
    slots = m.slots(table, b.iota((cfg.batch,), 0), pos, live)
    lengths = b.select(live, b.add(pos, b.scalar_like(1, pos)), b.scalar_like(0, pos))
    out, x, pools = m.blocks(tokens, pos, slots, pools,
                             lambda q, k, v, kp, vp: b.paged_attention(q, kp, vp, table, lengths))
    h, _ = b.add_rms_norm(out, x, m.w["final_norm"], cfg.model.eps)
    return b.build(m.answer(h, None) + pools)


def prefill_program(cfg: PagedConfig) -> str:
    b = Builder("jit_paged_prefill")
    m = _Model(b, cfg)
    n = cfg.chunk
    tokens, targets, count = b.param((n,), "s32"), b.param((n,), "s32"), b.param((), "s32")
    table = b.param((1, cfg.table_width), "s32")
    pools = m.pools()
    pos = b.iota((n,), 0)
    live = b.compare("LT", pos, b.broadcast_in_dim(count, (n,), []))
    slots = m.slots(table, b.scalar_like(0, pos), pos, live)

    def attend(q, k, v, kp, vp):  # the prompt's own keys: causal, from position 0
        rows = [b.reshape(t, (1, *t.shape)) for t in (q, k, v)]
        return b.custom_call(SDPA, [*rows, b.constant(0, "s32")], rows[0].shape, "bf16")

    out, x, pools = m.blocks(tokens, pos, slots, pools, attend)
    h, _ = b.add_rms_norm(out, x, m.w["final_norm"], cfg.model.eps)
    logits = m.mm(h, m.w["lm_head"])
    last = b.dynamic_slice(logits, [b.subtract(count, b.constant(1, "s32")), b.constant(0, "s32")],
                           (1, cfg.model.vocab))
    _, tok = b.argmax(last, 1, "s32")
    return b.build([tok, last, *m.scores(logits, targets)] + pools)


class PagedRunner:
    """Greedy serving: prompts join and leave between steps, each step decodes
    one token of every sequence. Pages are handed out from a free list as
    sequences grow."""

    def __init__(self, client, cfg: PagedConfig, weights: list[np.ndarray]):
        self.client, self.cfg = client, cfg
        self.prefill = client.compile(prefill_program(cfg))
        self.decode = client.compile(decode_program(cfg))
        self.weights = [client.buffer(w, "bf16") for w in weights]
        zero = np.zeros(cfg.pool_shape, np.uint16)
        self.pools = [client.buffer(zero, "bf16") for _ in range(2 * cfg.model.layers)]
        self.free = list(range(cfg.pages - 1, -1, -1))
        self.table = np.full((cfg.batch, cfg.table_width), -1, np.int32)
        self.length = np.full(cfg.batch, -1, np.int64)  # keys held; -1: an empty place
        self.token = np.zeros(cfg.batch, np.int32)

    def _hold(self, place: int, keys: int) -> None:
        """Pages for `keys` keys of the sequence at `place`, or none."""
        need = [i for i in range(-(-keys // self.cfg.page_size)) if self.table[place, i] < 0]
        if len(need) > len(self.free):
            raise MemoryError("no free page")
        for i in need:
            self.table[place, i] = self.free.pop()

    def _run(self, exe, args):
        outs = exe.execute_buffers(self.weights + [self.client.buffer(a) for a in args] + self.pools)
        self.pools = outs[6:]
        return [o.to_numpy() for o in outs[:6]]

    def add(self, prompt: np.ndarray):
        """Prefills a prompt at an empty place. Returns the place, the first
        generated token, its logits, and the prompt's scores: the log
        probability of each token but the first after those before it."""
        n = len(prompt)
        most = min(self.cfg.chunk, self.cfg.model.max_len)
        if not 1 <= n <= most:
            raise ValueError(f"a prompt has 1 to {most} tokens")
        places = np.flatnonzero(self.length < 0)
        if not len(places):
            raise ValueError("no empty place")
        place = int(places[0])
        self._hold(place, n)
        tokens, targets = np.zeros(self.cfg.chunk, np.int32), np.full(self.cfg.chunk, -1, np.int32)
        tokens[:n], targets[:n - 1] = prompt, prompt[1:]
        tok, logits, lp, *_ = self._run(self.prefill, [tokens, targets, np.array(n, np.int32), self.table[place:place + 1]])
        self.length[place], self.token[place] = n, tok[0]
        return place, int(tok[0]), logits[0], lp[:n - 1]

    def step(self):
        """One token for every sequence. Returns (places, tokens, logits, log
        probabilities, entropies, likeliest log probabilities and ids)."""
        places = np.flatnonzero(self.length >= 0)
        for p in places:
            if self.length[p] >= self.cfg.model.max_len:
                raise ValueError(f"the sequence at place {p} has max_len keys")
            self._hold(int(p), int(self.length[p]) + 1)
        outs = self._run(self.decode, [self.token, self.length.astype(np.int32), self.table])
        self.length[places] += 1
        self.token[places] = outs[0][places]
        return [places] + [o[places] for o in outs]

    def leave(self, place: int) -> None:
        """Takes a sequence out; its pages are free again."""
        self.free += [int(p) for p in self.table[place] if p >= 0]
        self.table[place] = -1
        self.length[place] = -1
