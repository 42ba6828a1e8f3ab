"""The operators in a run together: serving with pjrtx_amd/paged_llama.py, and
the end of a training step (programs.lm_head_loss), against the decoder's numpy
oracle and float64."""
import dataclasses
import json

import numpy as np
import pytest

from oracle import llama as O
from oracle import operators as P
from oracle import ops
from pjrtx_amd import llama_like as L
from pjrtx_amd import paged_llama as G
from pjrtx_amd import programs

pytestmark = pytest.mark.gpu

TOL = 2e-2  # of the logits' range: bf16 activations, as in test_gpu_llama.py
CFG = G.PagedConfig(model=L.TINY, kv_heads=2, batch=4, page_size=8, pages=20, chunk=16, top_k=3)


def weights(cfg, seed=0):
    """llama_like's weights with wk and wv of kv_heads, and the same for the
    oracle's model, whose heads each have their own keys: repeated."""
    full = L.init_weights(cfg.model, seed)
    names = [n for n, _ in L.weight_shapes(cfg.model)]
    m, kv = cfg.model, cfg.kv_heads * cfg.model.head_dim
    mine, dense = [], []
    for n, w in zip(names, full):
        if n.endswith(("wk", "wv")):
            w = np.ascontiguousarray(w[:, :kv])
            mine.append(w)
            r = w.reshape(m.d_model, cfg.kv_heads, m.head_dim).repeat(m.heads // cfg.kv_heads, 1)
            dense.append(np.ascontiguousarray(r.reshape(m.d_model, m.qdim)))
        else:
            mine.append(w)
            dense.append(w)
    assert [w.shape for w in mine] == [s for _, s in G.weight_shapes(cfg)]
    return mine, O.weights_f32(m, dense)


class Reference:
    """One sequence in the oracle's dense decoder."""

    def __init__(self, cfg, W, prompt):
        self.m, self.W = cfg.model, W
        self.k, self.v = O.empty_caches(cfg.model)
        self.n = len(prompt)
        self.logits = O.forward(self.m, W, prompt, 0, self.k, self.v)[1]

    def next(self, token):
        self.logits = O.forward(self.m, self.W, np.array([token], np.int32), self.n, self.k, self.v)[1]
        self.n += 1


def near(got, want):
    scale = float(np.abs(want).max())
    assert np.abs(ops.bf16_bits_to_f32(got) - want).max() <= TOL * scale
    return scale


def test_serving_sequences_that_join_and_leave(client):
    mine, W = weights(CFG)
    run = G.PagedRunner(client, CFG, mine)
    rng = np.random.default_rng(1)
    ref = {}

    def join(n):
        prompt = rng.integers(0, CFG.model.vocab, n).astype(np.int32)
        place, tok, logits, scores = run.add(prompt)
        ref[place] = Reference(CFG, W, prompt)
        near(logits, ref[place].logits)
        assert tok == int(np.argmax(ops.bf16_bits_to_f32(logits)))
        # the prompt's scores: each from the oracle's logits of its prefix,
        # which may be TOL of the range off, at the token and in the lse
        for i in range(1, n):
            want = Reference(CFG, W, prompt[:i]).logits.astype(np.float64)
            lp = P.token_logprobs(want[None], prompt[i:i + 1])[0][0]
            assert abs(scores[i - 1] - lp) <= 2 * TOL * np.abs(want).max()
        return place

    def step():
        fed = run.token.copy()
        places, tok, logits, lp, entropy, top, ids = run.step()
        assert sorted(places) == sorted(ref)
        for j, p in enumerate(places):
            ref[p].next(int(fed[p]))
            near(logits[j], ref[p].logits)
            # the scores belong to the logits that were returned
            x = ops.bf16_bits_to_f32(logits[j]).astype(np.float64)[None]
            wlp, went, _, wtop, wids = P.token_logprobs(x, tok[j:j + 1], CFG.top_k)
            assert tok[j] == int(np.argmax(x)) == ids[j, 0] and np.array_equal(ids[j], wids[0])
            np.testing.assert_allclose([lp[j], entropy[j], *top[j]], [wlp[0], went[0], *wtop[0]], atol=1e-5)

    a, b = join(5), join(1)
    for _ in range(6):
        step()
    c = join(16)              # two whole pages
    for _ in range(3):
        step()
    run.leave(b)
    del ref[b]
    step()
    d = join(9)               # in the place and pages of the one that left
    assert d == b
    for _ in range(8):
        step()
    assert len({p for p in run.table.ravel() if p >= 0}) == (run.table >= 0).sum() == CFG.pages - len(run.free)
    for p in (a, c, d):
        run.leave(p)
    assert len(run.free) == CFG.pages


def test_pages_of_other_sequences_are_left_as_they_were(client):
    mine, _ = weights(CFG)
    run = G.PagedRunner(client, CFG, mine)
    place = run.add(np.arange(10, dtype=np.int32))[0]
    before = [p.to_numpy() for p in run.pools]
    held = set(run.table[place][run.table[place] >= 0])
    run.step()
    page, pos = run.table[place, 10 // 8], 10 % 8
    for x, y in zip(before, run.pools):
        y = y.to_numpy()
        changed = {tuple(i) for i in np.argwhere((x != y).any(-1))}
        assert changed <= {(page, h, pos) for h in range(CFG.kv_heads)} and changed
        assert not y[[p for p in range(CFG.pages) if p not in held]].any()


def test_the_caches_are_written_in_place(client):
    plan = json.loads(client.compile(G.decode_program(CFG)).optimized_program())
    kinds = [s["library"] for s in plan["steps"] if s["kind"] == "library"]
    n = CFG.model.layers
    assert kinds.count("paged_attention") == n and kinds.count("token_logprobs") == 1
    assert kinds.count("add_rms_norm") == 2 * n + 1
    appends = [s for s in plan["steps"] if s.get("library") == "paged_append"]
    assert [s["in_place_operands"] for s in appends] == [3] * n and len(plan["written_params"]) == 2 * n


def test_a_captured_step_replays_like_an_eager_one(client, run_fresh):
    """The decode step is launch-bound at this size and replays from a captured
    graph after two calls: every replay against the oracle, with lengths that
    change from call to call and other programs between."""
    cfg = dataclasses.replace(CFG, batch=2)
    mine, W = weights(cfg, seed=3)
    run = G.PagedRunner(client, cfg, mine)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, cfg.model.vocab, n).astype(np.int32) for n in (3, 11)]
    ref = {}
    for p in prompts:
        place = run.add(p)[0]
        ref[place] = Reference(cfg, W, p)
    for i in range(12):
        fed = run.token.copy()
        places, _, logits, *_ = run.step()
        for j, p in enumerate(places):
            ref[p].next(int(fed[p]))
            near(logits[j], ref[p].logits)
        if i % 4 == 3:
            client.compile(programs.topk_logits(2, 100, 3))(np.zeros((2, 100), np.uint16), dtypes=["bf16"])
    assert run.decode.graph_stats()["replays"] > 0


def test_prompts_that_find_no_room_take_nothing(client):
    cfg = dataclasses.replace(CFG, pages=3, chunk=64)
    run = G.PagedRunner(client, cfg, weights(cfg)[0])
    run.add(np.arange(16, dtype=np.int32))
    with pytest.raises(MemoryError):
        run.add(np.arange(9, dtype=np.int32))
    with pytest.raises(ValueError, match="1 to 40"):
        run.add(np.zeros(41, np.int32))
    assert len(run.free) == 1 and (run.table[1:] < 0).all() and (run.length >= 0).sum() == 1
    run.step()
    assert not run.free
    run.leave(0)
    assert sorted(run.free) == [0, 1, 2]


def test_a_loss_of_no_rows_is_zero(client):
    rng = np.random.default_rng(6)
    args = [ops.f32_to_bf16_bits(rng.standard_normal(s).astype(np.float32)) for s in ((5, 64), (5, 64), (64,), (64, 100))]
    tok = np.array([-1, 100, -7, 2 ** 31 - 1, -2 ** 31], np.int32)
    loss, *grads = client.compile(programs.lm_head_loss(5, 64, 100, 0.1))(*args, tok, dtypes=["bf16"] * 4 + [None])
    assert loss == 0 and all((ops.bf16_bits_to_f32(g) == 0).all() for g in grads)


@pytest.mark.parametrize("weight", [0.0, 0.1])
def test_rows_left_out_of_the_loss_may_hold_anything(client, weight):
    """Rows without a target, of NaN, infinities and numbers beyond bf16: the
    loss and the gradients are those of the same rows at zero, and their own
    gradient is zero."""
    rng = np.random.default_rng(8)
    bf = lambda a: ops.f32_to_bf16_bits(np.asarray(a, np.float32))  # noqa: E731
    x, res = rng.standard_normal((2, 9, 64))
    g, w = bf(1 + 0.1 * rng.standard_normal(64)), bf(rng.standard_normal((64, 100)) * 0.125)
    tok = rng.integers(0, 100, 9).astype(np.int32)
    out = [1, 4, 6, 8]
    tok[out] = [-1, 100, -1, -5]
    exe = client.compile(programs.lm_head_loss(9, 64, 100, weight))
    x[out] = res[out] = 0
    want = exe(bf(x), bf(res), g, w, tok, dtypes=["bf16"] * 4 + [None])
    x[1, 3], x[4], res[6], x[8] = np.nan, np.inf, -np.inf, 3e38
    res[8] = 3e38
    got = exe(bf(x), bf(res), g, w, tok, dtypes=["bf16"] * 4 + [None])
    assert np.isfinite(want[0])
    for a, b in zip(got, want):
        assert a.tobytes() == b.tobytes()
    assert (ops.bf16_bits_to_f32(got[1][out]) == 0).all()


@pytest.mark.parametrize("rows,d,vocab,weight", [(1, 64, 100, 0.0), (7, 96, 333, 0.1), (130, 128, 1000, 0.0)])
def test_loss_and_gradients(client, rows, d, vocab, weight):
    """Each result against float64 on the same inputs. The bf16 roundings on
    the way: of h (2^-8 of it, which the logits' error is a d-sum of), of the
    logits (2^-8), of d logits and of d h. Bounds are sums of these over the
    products' magnitudes."""
    u = 2.0 ** -8
    rng = np.random.default_rng(rows)
    bf = lambda x: ops.f32_to_bf16_bits(np.asarray(x, np.float32))  # noqa: E731
    f = lambda a: ops.bf16_bits_to_f32(a).astype(np.float64)  # noqa: E731
    x, res = bf(rng.standard_normal((rows, d))), bf(rng.standard_normal((rows, d)))
    g, w = bf(1 + 0.1 * rng.standard_normal(d)), bf(rng.standard_normal((d, vocab)) * d ** -0.5)
    tok = rng.integers(0, vocab, rows).astype(np.int32)
    if rows > 3:
        tok[[1, 3]] = [-1, vocab]  # rows that are not counted
    loss, dx, dg, dw = client.compile(programs.lm_head_loss(rows, d, vocab, weight))(x, res, g, w, tok,
                                                                                    dtypes=["bf16"] * 4 + [None])
    h, t = P.add_rms_norm(f(x), f(res), f(g), 1e-5)
    logits = h @ f(w)
    lp, H, lse = P.token_logprobs(logits, tok)
    share = ((tok >= 0) & (tok < vocab)) / max(1, ((tok >= 0) & (tok < vocab)).sum())
    want = -(share * (lp + weight * H)).sum()
    dl = P.token_logprobs_grad(logits, tok, lse, H, -share, -weight * share)
    dh = dl @ f(w).T
    wx, wg = P.add_rms_norm_grad(dh, None, t, f(g), 1e-5)
    ww = h.T @ dl
    e_logit = u * (np.abs(h) @ np.abs(f(w)) + np.abs(logits)) * 1.1        # of each logit
    most = e_logit.max()
    assert abs(loss - want) <= (2 + 4 * weight * (1 + H.max())) * most + 1e-5
    # p is off by 2 e_logit of itself, and d logits is rounded
    p = np.exp(logits - lse[:, None])
    e_dl = share[:, None] * p * (1 + weight * (1 + np.abs(logits - lse[:, None]) + H[:, None])) * 4 * most + u * np.abs(dl)
    e_dh = e_dl @ np.abs(f(w)).T + 2 * u * np.abs(dh)
    r = 1 / np.sqrt((t * t).mean(1, keepdims=True) + 1e-5)
    n = np.abs(t) * r
    e_dn = e_dh * np.abs(f(g)) + 2 * u * np.abs(dh * f(g))
    e_dx = r * (e_dn + n * (e_dn * n).mean(1, keepdims=True)) + 3 * u * (np.abs(wx) + r * n * np.abs((dh * f(g) * n).mean(1, keepdims=True)))
    assert (np.abs(f(dx) - wx) <= e_dx + 1e-12).all()
    assert (np.abs(f(dg) - wg) <= (e_dh * n + 2 * u * np.abs(dh) * n).sum(0) + u * np.abs(wg) + 1e-12).all()
    assert (np.abs(f(dw) - ww) <= u * (np.abs(h).T @ np.abs(dl)) * 1.1 + np.abs(h).T @ e_dl + u * np.abs(ww) + 1e-12).all()
