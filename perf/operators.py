"""The operators of a decoder's serving and training step that the plugin
offers as custom calls, as cases that can be timed and checked:

  attention  one new token a sequence over a paged key-value cache
  append     new keys and values written into the cache's pages
  norm       the residual's addition with the root-mean-square norm, its
             result in the input's type or in 8 bits with a scale a row
  norm_grad  that norm's gradient: the input's, and the gain's over all rows
  logprobs   log probabilities of given tokens, with the distribution's
             entropy and the likeliest tokens
  logprobs_grad  the gradient of log probabilities and entropies

`prepare` makes a case's inputs on the GPU and, for the plugin's kernels,
compiles the program that makes the call; `run` is one pass on them: torch
operations, or one execute on the tensors' memory. A sequence's lengths go by
the case, so that `work` knows them; the seed orders them.
"""
import math

import torch

own = False

_TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "s32": torch.int32, "s8": torch.int8}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------- cases

def listed():
    return [
        # One sequence of the benchmark's decoder, 16 heads: the smallest
        # call, a few microseconds, where launch and latency count.
        {"name": "attention_1x600", "kind": "attention", "batch": 1, "kv_heads": 16, "group": 1, "head_dim": 128,
         "max_len": 600, "ragged": False, "page": 16, "window": 0, "dtype": "bf16"},
        # A batch being served: grouped heads, lengths from 32 to 4064.
        {"name": "attention_64x4096_ragged", "kind": "attention", "batch": 64, "kv_heads": 8, "group": 4,
         "head_dim": 128, "max_len": 4096, "ragged": True, "page": 16, "window": 0, "dtype": "bf16"},
        # Two long documents: few rows, so the length has to be split.
        {"name": "attention_2x131072", "kind": "attention", "batch": 2, "kv_heads": 4, "group": 8, "head_dim": 128,
         "max_len": 131072, "ragged": False, "page": 64, "window": 0, "dtype": "f16"},
        # 32-bit, an odd batch, pages and heads that are no power of two, a
        # sliding window.
        {"name": "attention_7x1500_f32", "kind": "attention", "batch": 7, "kv_heads": 3, "group": 4, "head_dim": 96,
         "max_len": 1500, "ragged": True, "page": 24, "window": 1000, "dtype": "f32"},
        # One token of each of 64 sequences.
        {"name": "append_64", "kind": "append", "tokens": 64, "kv_heads": 8, "head_dim": 128, "page": 16, "pages": 4096,
         "dtype": "bf16"},
        # A prompt's chunk, the batch padded.
        {"name": "append_8000", "kind": "append", "tokens": 8000, "kv_heads": 8, "head_dim": 128, "page": 16,
         "pages": 2048, "dtype": "f16"},
        # One token's row in the benchmark's decoder.
        {"name": "norm_1x2048", "kind": "norm", "rows": 1, "dim": 2048, "quantize": False, "dtype": "bf16"},
        # A prefill's rows for a product in 8 bits.
        {"name": "norm_8192x4096_s8", "kind": "norm", "rows": 8192, "dim": 4096, "quantize": True, "dtype": "bf16"},
        # A training step's rows; their count is no multiple of a tile.
        {"name": "norm_grad_8000x2048", "kind": "norm_grad", "rows": 8000, "dim": 2048, "dtype": "bf16"},
        # Sampling's answer for a batch: the largest vocabulary here.
        {"name": "logprobs_64x128256", "kind": "logprobs", "rows": 64, "vocab": 128256, "top_k": 20, "dtype": "bf16"},
        # A prompt scored in 32 bits.
        {"name": "logprobs_1000x32000_f32", "kind": "logprobs", "rows": 1000, "vocab": 32000, "top_k": 5,
         "dtype": "f32"},
        # A training step's loss gradient.
        {"name": "logprobs_grad_2000x32000", "kind": "logprobs_grad", "rows": 2000, "vocab": 32000, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    """An integer in [lo, hi], spread over its logarithm; half of them round."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v >= 64 and rng.random() < 0.5:
        v = v // 64 * 64
    return max(lo, min(hi, v))


_MOST = 550_000_000  # bytes of a drawn case's work: the largest listed one's


def draw(rng):
    kind = rng.choice(["attention", "attention", "append", "norm", "norm_grad", "logprobs", "logprobs_grad"])
    while True:
        c = _draw(kind, rng)
        if work(c)["bytes"] <= _MOST and _held(c) <= 4 * _MOST:
            return c


def _draw(kind, rng):
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "attention":
        max_len = _log_int(rng, 1, 131072)
        return {"kind": kind, "batch": _log_int(rng, 1, 128), "kv_heads": rng.choice([1, 2, 3, 4, 8, 16]),
                "group": rng.choice([1, 1, 2, 4, 5, 8, 16, 32]), "head_dim": rng.choice([64, 96, 128, 128, 256]),
                "max_len": max_len, "ragged": rng.random() < 0.6, "page": rng.choice([8, 16, 16, 24, 32, 64, 128]),
                "window": rng.choice([0, 0, 0, max(1, max_len // 3)]), "dtype": dtype}
    if kind == "append":
        return {"kind": kind, "tokens": _log_int(rng, 1, 8192), "kv_heads": rng.choice([1, 2, 3, 4, 8, 16]),
                "head_dim": rng.choice([64, 80, 96, 128, 256]), "page": rng.choice([8, 16, 24, 32, 64]),
                "pages": 2048, "dtype": dtype}
    if kind == "norm":
        return {"kind": kind, "rows": _log_int(rng, 1, 16384), "dim": _log_int(rng, 64, 16384),
                "quantize": rng.random() < 0.4, "dtype": dtype}
    if kind == "norm_grad":
        return {"kind": kind, "rows": _log_int(rng, 1, 16384), "dim": _log_int(rng, 64, 16384), "dtype": dtype}
    c = {"kind": kind, "rows": _log_int(rng, 1, 4096), "vocab": _log_int(rng, 1000, 256000), "dtype": dtype}
    if kind == "logprobs":
        c["top_k"] = rng.choice([0, 1, 5, 20])
    return c


def _held(c):
    """Bytes of a case's largest buffer."""
    if c["kind"] == "attention":
        return _pages(c) * c["page"] * c["kv_heads"] * c["head_dim"] * _SIZE[c["dtype"]]
    if c["kind"] == "append":
        return c["pages"] * c["page"] * c["kv_heads"] * c["head_dim"] * _SIZE[c["dtype"]]
    return c["rows"] * c.get("vocab", c.get("dim")) * _SIZE[c["dtype"]]


def _lengths(c):
    """Each sequence's length: all the same, or spread evenly up to max_len."""
    b, n = c["batch"], c["max_len"]
    return [n * (2 * i + 1) // (2 * b) for i in range(b)] if c["ragged"] else [n] * b


def _pages(c):
    return sum(-(-n // c["page"]) for n in _lengths(c)) + 8  # and some that no sequence has


def _attended(c):
    return [min(n, c["window"]) if c["window"] else n for n in _lengths(c)]


def work(case):
    c, kind = case, case["kind"]
    e = _SIZE[c["dtype"]]
    if kind == "attention":
        keys = sum(_attended(c))
        row = c["kv_heads"] * c["head_dim"]
        q = c["batch"] * row * c["group"]
        return {"bytes": e * (2 * keys * row + 2 * q) + 4 * (c["batch"] + sum(-(-n // c["page"]) for n in _attended(c))),
                "flops": 4 * keys * row * c["group"]}
    if kind == "append":
        n = c["tokens"]
        return {"bytes": n * (4 * e * c["kv_heads"] * c["head_dim"] + 4), "flops": 0}
    if kind in ("norm", "norm_grad"):
        n = c["rows"] * c["dim"]
        if kind == "norm":  # x and the residual in; the sum and the norm out
            return {"bytes": e * (4 * n + c["dim"]) + 4 * c["rows"] * c["quantize"], "flops": 6 * n}
        return {"bytes": e * (4 * n + 2 * c["dim"]), "flops": 12 * n}
    n = c["rows"] * c["vocab"]
    if kind == "logprobs":
        return {"bytes": e * n + c["rows"] * (16 + 8 * c["top_k"]), "flops": 6 * n}
    return {"bytes": 2 * e * n + 20 * c["rows"], "flops": 8 * n}


# ------------------------------------------------------------------ inputs

def _inputs(c, seed):
    """The arguments of the call, in its order, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = c["kind"]

    def normal(shape, scale=1.0, dtype=None):
        return torch.randn(shape, device="cuda", generator=g).mul_(scale).to(_TORCH[dtype or c["dtype"]])

    def shuffled(n):
        return torch.randperm(n, device="cuda", generator=g)

    if kind == "attention":
        lengths = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda")[shuffled(c["batch"])]
        page, pool = c["page"], _pages(c)
        kv = (pool, c["kv_heads"], page, c["head_dim"])
        # Each sequence's pages lie anywhere in the pool; entries past its
        # last page name none.
        used = (lengths.long() + page - 1) // page
        width = -(-c["max_len"] // page) + 1
        at = torch.arange(width, device="cuda")
        first = torch.cumsum(used, 0) - used
        table = shuffled(pool)[(first[:, None] + at).clamp(max=pool - 1)].int()
        table = torch.where(at < used[:, None], table, torch.full_like(table, -1))
        return [normal((c["batch"], c["kv_heads"] * c["group"], c["head_dim"])), normal(kv), normal(kv), table, lengths]
    if kind == "append":
        n = c["tokens"]
        kv = (c["pages"], c["kv_heads"], c["page"], c["head_dim"])
        new = (n, c["kv_heads"], c["head_dim"])
        slots = shuffled(c["pages"] * c["page"])[:n].int()
        if n >= 16:  # padding rows name no slot
            slots[shuffled(n)[:n // 16]] = -1
        return [normal(kv), normal(kv), normal(new), normal(new), slots]
    if kind == "norm":
        shape = (c["rows"], c["dim"])
        return [normal(shape), normal(shape, 3.0), 1 + normal((c["dim"],), 0.1, "f32").to(_TORCH[c["dtype"]])]
    if kind == "norm_grad":
        shape = (c["rows"], c["dim"])
        return [normal(shape, 0.1), normal(shape, 0.1), normal(shape, 3.0),
                1 + normal((c["dim"],), 0.1, "f32").to(_TORCH[c["dtype"]])]
    logits = normal((c["rows"], c["vocab"]), 3.0)
    tokens = torch.randint(0, c["vocab"], (c["rows"],), device="cuda", generator=g, dtype=torch.int32)
    if kind == "logprobs":
        return [logits, tokens]
    # What the forward call gave, and the loss's gradients of its results.
    x = logits.float()
    lse = torch.logsumexp(x, 1)
    logp = x - lse[:, None]
    entropy = -(logp.exp() * logp).sum(1)
    return [logits, tokens, lse, entropy, normal((c["rows"],), 1.0, "f32"), normal((c["rows"],), 0.01, "f32")]


def _results(c):
    """Shape and type of each result."""
    kind, t = c["kind"], c["dtype"]
    if kind == "attention":
        return [((c["batch"], c["kv_heads"] * c["group"], c["head_dim"]), t)]
    if kind == "norm":
        shape = (c["rows"], c["dim"])
        return [(shape, t), ((c["rows"],), "f32"), (shape, t)] if c["quantize"] else [(shape, t), (shape, t)]
    if kind == "norm_grad":
        return [((c["rows"], c["dim"]), t), ((c["dim"],), t)]
    if kind == "logprobs":
        r, k = (c["rows"],), (c["rows"], c["top_k"])
        return [(r, "f32")] * 3 + ([(k, "f32"), (k, "s32")] if c["top_k"] else [])
    return [((c["rows"], c["vocab"]), t)]


_EPS = 1e-5
_client = None


def _program(c, inputs):
    """The program that makes the case's call."""
    from pjrtx_amd.hlo import Builder
    names = {v: k for k, v in _TORCH.items()}
    kind = c["kind"]
    b = Builder("jit_" + kind)
    p = [b.param(tuple(x.shape), names[x.dtype], donate=kind == "append" and i < 2) for i, x in enumerate(inputs)]
    if kind == "attention":
        out = [b.paged_attention(*p, window=c["window"])]
    elif kind == "append":
        out = list(b.paged_append(*p))
    elif kind == "norm" and c["quantize"]:
        # The next operator's view of the 8-bit rows: the values they stand for.
        # The rows themselves are a result too, in the caller's memory: as a value
        # between the two steps they could be more than the 64 MiB that such a
        # call has for all of them.
        y8, scale, total = b.add_rms_norm(*p, eps=_EPS, quantize=True)
        y = b.multiply(b.convert(y8, "f32"), b.broadcast_in_dim(scale, y8.shape, [0]))
        out = [b.convert(y, c["dtype"]), scale, total, y8]
    elif kind == "norm":
        out = list(b.add_rms_norm(*p, eps=_EPS))
    elif kind == "norm_grad":
        out = list(b.add_rms_norm_grad(*p, eps=_EPS))
    elif kind == "logprobs":
        out = list(b.token_logprobs(*p, top_k=c["top_k"]))
    else:
        out = [b.token_logprobs_grad(*p)]
    return b.build(out)


def _compiled(c, inputs):
    """That program, loaded."""
    global _client
    from pjrtx_amd.pjrt import Client
    if _client is None:
        _client = Client()
    return _client.compile(_program(c, inputs))


def prepare(case, seed):
    inputs = _inputs(case, seed)
    state = {"case": case, "inputs": inputs}
    if own:
        # The handle, and the memory that the results go to; the cache's pages
        # are written where they are.
        state["exe"] = _compiled(case, inputs)
        state["out"] = inputs[:2] if case["kind"] == "append" else [
            torch.empty(shape, dtype=_TORCH[t], device="cuda") for shape, t in _results(case)]
        state["in_ptrs"] = [x.data_ptr() for x in inputs]
        held = []
        if case["kind"] == "norm" and case["quantize"]:
            held = [torch.empty((case["rows"], case["dim"]), dtype=torch.int8, device="cuda")]
        state["held"] = held
        state["out_ptrs"] = [x.data_ptr() for x in state["out"] + held]
    return state


def run(state):
    if own:
        state["exe"].execute_noalloc(state["in_ptrs"], state["out_ptrs"])
        return state["out"]
    return _PLAIN[state["case"]["kind"]](state["case"], *state["inputs"])


# -------------------------------------------------------------- plain forms

def _plain_attention(c, q, k_pages, v_pages, table, lengths):
    batch, kv_heads, head_dim = c["batch"], c["kv_heads"], c["head_dim"]
    at = table.clamp(min=0).long()
    k = k_pages[at].transpose(1, 2).reshape(batch, kv_heads, -1, head_dim).float()
    v = v_pages[at].transpose(1, 2).reshape(batch, kv_heads, -1, head_dim).float()
    s = torch.matmul(q.float().view(batch, kv_heads, c["group"], head_dim), k.transpose(2, 3)) / math.sqrt(head_dim)
    key = torch.arange(k.shape[2], device="cuda")
    seen = (key < lengths[:, None]) & (table >= 0).repeat_interleave(c["page"], 1)
    if c["window"]:
        seen &= key >= lengths[:, None] - c["window"]
    seen = seen[:, None, None]
    s = torch.where(seen, s, -math.inf)
    p = torch.where(seen, torch.exp(s - s.amax(3, keepdim=True)), 0.0)
    total = p.sum(3, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)  # a sequence of no keys answers zero
    return [out.reshape(q.shape).to(q.dtype)]


def _plain_append(c, k_pages, v_pages, k_new, v_new, slots):
    named = slots >= 0
    at = slots[named].long()
    page, slot = at // c["page"], at % c["page"]
    k_pages[page, :, slot] = k_new[named]
    v_pages[page, :, slot] = v_new[named]
    return [k_pages, v_pages]


def _plain_norm(c, x, residual, gain):
    s = x.float() + residual.float()
    y = s * torch.rsqrt((s * s).mean(1, keepdim=True) + _EPS) * gain.float()
    if not c["quantize"]:
        return [y.to(x.dtype), s.to(x.dtype)]
    scale = y.abs().amax(1) / 127
    y8 = torch.round(y / torch.where(scale > 0, scale, 1.0)[:, None]).to(torch.int8)
    return [(y8.float() * scale[:, None]).to(x.dtype), scale, s.to(x.dtype)]


def _plain_norm_grad(c, dy, dsum, s, gain):
    s, dy = s.float(), dy.float()
    r = torch.rsqrt((s * s).mean(1, keepdim=True) + _EPS)
    n, dn = s * r, dy * gain.float()
    dx = dsum.float() + r * (dn - n * (dn * n).mean(1, keepdim=True))
    return [dx.to(gain.dtype), (dy * n).sum(0).to(gain.dtype)]


def _plain_logprobs(c, logits, tokens):
    x = logits.float()
    shift = x.amax(1, keepdim=True)
    e = torch.exp(x - shift)
    total = e.sum(1)
    lse = shift[:, 0] + torch.log(total)
    entropy = torch.log(total) - (e * (x - shift)).sum(1) / total
    out = [x.gather(1, tokens.long()[:, None])[:, 0] - lse, entropy, lse]
    if c["top_k"]:
        # Ties go to the lowest index: ranked by the value's bits in order,
        # then by the index.
        bits = x.view(torch.int32).long()
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
        index = torch.arange(c["vocab"], device="cuda")
        top = torch.topk((order << 20) + (c["vocab"] - 1 - index), c["top_k"], dim=1)[0]
        top = c["vocab"] - 1 - (top & 0xFFFFF)
        out += [x.gather(1, top) - lse[:, None], top.int()]
    return out


def _plain_logprobs_grad(c, logits, tokens, lse, entropy, d_logprobs, d_entropy):
    logp = logits.float() - lse[:, None]
    p = torch.exp(logp)
    dx = -p * (d_logprobs[:, None] + d_entropy[:, None] * (logp + entropy[:, None]))
    dx.scatter_add_(1, tokens.long()[:, None], d_logprobs[:, None])
    return [dx.to(logits.dtype)]


_PLAIN = {"attention": _plain_attention, "append": _plain_append, "norm": _plain_norm, "norm_grad": _plain_norm_grad,
          "logprobs": _plain_logprobs, "logprobs_grad": _plain_logprobs_grad}


# -------------------------------------------------------------------- exact

def exact(case, seed):
    c, kind = case, case["kind"]
    if kind == "append":
        return None  # rows of the input, in another place
    a = _inputs(c, seed)
    if kind == "attention":
        q, k_pages, v_pages, table, lengths = a
        out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        for i, n in enumerate(lengths.tolist()):
            lo = max(0, n - c["window"]) if c["window"] else 0
            if n == lo:
                continue
            pages = table[i, : -(-n // c["page"])].long()
            for h in range(c["kv_heads"]):
                k, v = (x[pages, h].reshape(-1, c["head_dim"])[lo:n].double() for x in (k_pages, v_pages))
                heads = slice(h * c["group"], (h + 1) * c["group"])
                out[i, heads] = torch.softmax(q[i, heads].double() @ k.t() * c["head_dim"] ** -0.5, 1) @ v
        return [out]
    x = [t.double() if t.is_floating_point() else t.long() for t in a]
    if kind == "norm":
        s = x[0] + x[1]
        y = s / torch.sqrt(torch.linalg.vector_norm(s, dim=1, keepdim=True) ** 2 / c["dim"] + _EPS) * x[2]
        if not c["quantize"]:
            return [y, s]
        scale = torch.linalg.vector_norm(y, ord=math.inf, dim=1) / 127
        return [torch.floor(y / scale[:, None] + 0.5) * scale[:, None], scale, s]
    if kind == "norm_grad":
        dy, dsum, s, gain = x
        norm = torch.sqrt(torch.linalg.vector_norm(s, dim=1, keepdim=True) ** 2 / c["dim"] + _EPS)
        along = ((dy * gain * s).sum(1, keepdim=True) / c["dim"]) / norm ** 3
        return [dsum + dy * gain / norm - s * along, (dy * s / norm).sum(0)]
    rows = torch.arange(c["rows"], device="cuda")
    if kind == "logprobs":
        logp = torch.log_softmax(x[0], 1)
        got = [logp[rows, x[1]], torch.special.entr(logp.exp()).sum(1), torch.logsumexp(x[0], 1)]
        if c["top_k"]:
            got += [torch.sort(logp, dim=1, descending=True)[0][:, : c["top_k"]], None]
        return got
    logits, tokens, lse, entropy, d_logprobs, d_entropy = x
    p = torch.exp(logits - lse[:, None])
    dx = -p * d_logprobs[:, None] + d_entropy[:, None] * (torch.special.entr(p) - p * entropy[:, None])
    dx[rows, tokens] += d_logprobs
    return [dx]
