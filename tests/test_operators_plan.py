"""Lowering, refusals and plans of the operator custom calls (no GPU)."""
import json
import re

import numpy as np
import pytest

from pjrtx_amd.hlo import Builder
from pjrtx_amd.pjrt import PjrtError

INVALID, UNIMPLEMENTED = 3, 12
PAGES = (8, 2, 16, 64)


def plan(plugin, text):
    return json.loads(plugin.plan_json(text))


# operands (shape, dtype) and results of a call that is right, by target
CALLS = {
    "pjrtx.paged_attention": ([((3, 4, 64), "bf16"), (PAGES, "bf16"), (PAGES, "bf16"), ((3, 5), "s32"), ((3,), "s32")],
                              [((3, 4, 64), "bf16")]),
    "pjrtx.paged_append": ([(PAGES, "f16"), (PAGES, "f16"), ((7, 2, 64), "f16"), ((7, 2, 64), "f16"), ((7,), "s64")],
                           [(PAGES, "f16"), (PAGES, "f16")]),
    "pjrtx.add_rms_norm": ([((3, 5, 96), "f32"), ((3, 5, 96), "f32"), ((96,), "f32")],
                           [((3, 5, 96), "s8"), ((3, 5), "f32"), ((3, 5, 96), "f32")]),
    "pjrtx.add_rms_norm_grad": ([((5, 96), "f16")] * 3 + [((96,), "f16")], [((5, 96), "f16"), ((96,), "f16")]),
    "pjrtx.token_logprobs": ([((6, 50), "bf16"), ((6,), "s32")],
                             [((6,), "f32")] * 3 + [((6, 4), "f32"), ((6, 4), "s32")]),
    "pjrtx.token_logprobs_grad": ([((6, 50), "f32"), ((6,), "s64")] + [((6,), "f32")] * 4, [((6, 50), "f32")]),
}


def text_of(target, ins, outs, config=None):
    b = Builder()
    return b.build(b.operator_call(target, [b.param(*t) for t in ins], outs, config))


@pytest.mark.parametrize("target", CALLS)
def test_lowers_to_one_step(plugin, target):
    p = plan(plugin, text_of(target, *CALLS[target]))
    assert [s["library"] for s in p["steps"]] == [target.split(".")[1]]


def test_forms_of_the_norm(plugin):
    x, g = ((5, 96), "bf16"), ((96,), "bf16")
    for ins, outs in (([x, g], [x]), ([x, g], [((5, 96), "s8"), ((5,), "f32")]), ([x, x, g], [x, x]),
                      ([((96,), "bf16"), g], [((96,), "bf16")])):
        assert len(plan(plugin, text_of("pjrtx.add_rms_norm", ins, outs, {"eps": 1e-6}))["steps"]) == 1
    assert len(plan(plugin, text_of("pjrtx.add_rms_norm_grad", [x, x, g], [x, g]))["steps"]) == 1


def test_generic_form_and_empty_batches(plugin):
    ins, outs = CALLS["pjrtx.token_logprobs"]
    text = text_of("pjrtx.token_logprobs", ins, outs)
    types = ", ".join(t.split(": ")[1] for t in ("a: tensor<6x50xbf16>", "b: tensor<6xi32>"))
    line = next(s for s in text.splitlines() if "custom_call" in s)
    generic = ('    %0:5 = "stablehlo.custom_call"(%arg0, %arg1) <{api_version = 4 : i32, backend_config = {}, '
               'call_target_name = "pjrtx.token_logprobs"}> {mhlo.frontend_attributes = {}} : (' + types + ") -> "
               + line.split(" -> ")[1])
    assert plan(plugin, text.replace(line, generic))["steps"][0]["library"] == "token_logprobs"
    empty = {"pjrtx.paged_attention": {0: (0, 4, 64), 3: (0, 5), 4: (0,)}, "pjrtx.paged_append": {2: (0, 2, 64), 3: (0, 2, 64), 4: (0,)}}
    for target, shapes in empty.items():
        ins, outs = CALLS[target]
        ins = [(shapes.get(i, s), t) for i, (s, t) in enumerate(ins)]
        outs = [(shapes[0], outs[0][1])] if 0 in shapes else outs
        assert len(plan(plugin, text_of(target, ins, outs))["steps"]) == 1


def bad(target, operand=None, shape=None, dtype=None, result=None, config=None, drop=None, drop_result=False, code=INVALID):
    return target, operand, shape, dtype, result, config, drop, drop_result, code


ATT, APP, NORM, GRAD = "pjrtx.paged_attention", "pjrtx.paged_append", "pjrtx.add_rms_norm", "pjrtx.add_rms_norm_grad"
LOG, LGRAD = "pjrtx.token_logprobs", "pjrtx.token_logprobs_grad"


@pytest.mark.parametrize("case", [
    bad(ATT, drop=4), bad(ATT, 0, (3, 4)), bad(ATT, 0, (3, 3, 64)), bad(ATT, 0, (3, 4, 32)), bad(ATT, 0, dtype="f32"),
    bad(ATT, 1, (8, 2, 16, 32)), bad(ATT, 2, dtype="f16"), bad(ATT, 2, (8, 2, 8, 64)), bad(ATT, 3, dtype="s64"),
    bad(ATT, 3, (2, 5)), bad(ATT, 3, (3, 0)), bad(ATT, 4, (4,)), bad(ATT, 4, dtype="u32"),
    bad(ATT, result=(0, (3, 4, 64), "f32")), bad(ATT, config={"window": -1}), bad(ATT, config={"soft_cap": 1.0}),
    bad(ATT, config={"scale": float("inf")}), bad(ATT, config={"scale": float("nan")}), bad(ATT, 3, (3, 1 << 27), code=UNIMPLEMENTED),
    bad(APP, drop=4), bad(APP, 2, (7, 3, 64)), bad(APP, 3, (6, 2, 64)), bad(APP, 4, (6,)), bad(APP, 4, dtype="u32"),
    bad(APP, 3, dtype="f32"), bad(APP, result=(1, PAGES, "f32")), bad(APP, drop_result=True), bad(APP, config={"page": 16}),
    bad(NORM, 1, (3, 5, 64)), bad(NORM, 2, (64,)), bad(NORM, 2, dtype="f16"), bad(NORM, 0, dtype="s32"),
    bad(NORM, result=(1, (3, 4), "f32")), bad(NORM, result=(1, (3, 5), "bf16")), bad(NORM, result=(0, (3, 5, 96), "u8")),
    bad(NORM, drop_result=True), bad(NORM, config={"eps": -1e-5}), bad(NORM, config={"epsilon": 1e-5}), bad(NORM, drop=1),
    bad(GRAD, 1, dtype="f32"), bad(GRAD, 3, (95,)), bad(GRAD, result=(1, (96,), "f32")), bad(GRAD, drop_result=True),
    bad(LOG, 0, (6, 0)), bad(LOG, 0, dtype="s32"), bad(LOG, 1, (5,)), bad(LOG, 1, dtype="f32"),
    bad(LOG, result=(3, (6, 51), "f32")), bad(LOG, result=(4, (6, 4), "s64")), bad(LOG, result=(0, (6,), "bf16")),
    bad(LOG, drop_result=True), bad(LOG, config={"top_k": 4}),
    bad(LGRAD, 4, (5,)), bad(LGRAD, 2, dtype="bf16"), bad(LGRAD, drop=5), bad(LGRAD, result=(0, (6, 50), "bf16")),
], ids=str)
def test_refusals(plugin, case):
    target, operand, shape, dtype, result, config, drop, drop_result, code = case
    ins, outs = [list(x) for x in CALLS[target][0]], [list(x) for x in CALLS[target][1]]
    if operand is not None:
        ins[operand] = [shape or ins[operand][0], dtype or ins[operand][1]]
    if result:
        outs[result[0]] = list(result[1:])
    if drop is not None:
        del ins[drop]
    if drop_result:
        del outs[-1]
    with pytest.raises(PjrtError) as e:
        plan(plugin, text_of(target, ins, outs, config))
    assert e.value.code == code and target in e.value.message, e.value.message


def test_top_k_above_the_limit_and_head_dim(plugin):
    rows = [((6,), "f32")] * 3
    with pytest.raises(PjrtError) as e:
        plan(plugin, text_of(LOG, [((6, 500), "f32"), ((6,), "s32")], rows + [((6, 129), "f32"), ((6, 129), "s32")]))
    assert e.value.code == UNIMPLEMENTED
    pages = (8, 2, 16, 520)
    with pytest.raises(PjrtError) as e:
        plan(plugin, text_of(ATT, [((3, 4, 520), "f32"), (pages, "f32"), (pages, "f32"), ((3, 5), "s32"), ((3,), "s32")],
                             [((3, 4, 520), "f32")]))
    assert e.value.code == UNIMPLEMENTED


def _append(donate, read_after=False, same=False):
    b = Builder()
    k = b.param(PAGES, "bf16", donate=donate)
    v = k if same else b.param(PAGES, "bf16", donate=donate)
    new, slots = b.param((7, 2, 64), "bf16"), b.param((7,), "s32")
    k2, v2 = b.paged_append(k, v, new, new, slots)
    k3, v3 = b.paged_append(k2, v2, new, new, slots)
    out = [k3, v3]
    if read_after:
        out.append(b.add(k, k))
    return b.build(out)


def test_donated_pages_are_written_in_place(plugin):
    p = plan(plugin, _append(True))
    assert [s["in_place_operands"] for s in p["steps"]] == [3, 3] and sorted(p["written_params"]) == [0, 1]
    # the second call's operands die there whoever owns the first's
    p = plan(plugin, _append(False))
    assert [s["in_place_operands"] for s in p["steps"]] == [0, 3] and p["written_params"] == []


def test_one_value_for_keys_and_values_is_not_written_in_place(plugin):
    p = plan(plugin, _append(True, same=True))
    assert [s["in_place_operands"] for s in p["steps"]] == [0, 3]


def test_pages_read_later_are_kept(plugin):
    p = plan(plugin, _append(True, read_after=True))
    for i, s in enumerate(p["steps"]):
        if s.get("library") != "paged_append":
            continue
        later = [v for t in p["steps"][i + 1:] for v in t["inputs"]]
        for k in range(2):
            assert not (s["in_place_operands"] >> k & 1) or s["inputs"][k] not in later


def test_attributes_as_jax_prints_them(plugin):
    """Hexadecimal bits are infinities and NaNs; layouts, aliases and unknown
    attributes of the call itself are not the operator's."""
    ins, outs = CALLS[ATT]
    text = text_of(ATT, ins, outs, {"scale": 0.25, "window": 7})
    assert len(plan(plugin, text)["steps"]) == 1
    for value in ("1.0e39 : f64", "-1.0e300 : f64", "0x7F800000 : f32", "0xFFC00000 : f32", "true", '"1.0"', "[1.0]", "1.0.0 : f32"):
        with pytest.raises(PjrtError) as e:
            plan(plugin, text.replace("2.50000000000000000e-01 : f64", value))
        assert e.value.code == INVALID and "scale" in e.value.message
    for value in ("9.99999974E-6 : f32", "1 : i64", "0.5", "-2.0e+00 : f64"):
        assert plan(plugin, text.replace("2.50000000000000000e-01 : f64", value))["steps"]
    config = text[text.index("backend_config = {"):text.index("}", text.index("backend_config = {")) + 1]
    assert "scale" in config and "window" in config
    text = text.replace("window = 7", "window = -7")
    for form in (config, 'backend_config = "", mhlo.' + config, "mhlo." + config + ', backend_config = ""'):
        with pytest.raises(PjrtError) as e:
            plan(plugin, text.replace(config.replace("= 7", "= -7"), form.replace("= 7", "= -7")))
        assert "window" in e.value.message
    with pytest.raises(PjrtError) as e:
        plan(plugin, text.replace(config.replace("= 7", "= -7"), 'backend_config = "window=7"'))
    assert e.value.code == INVALID and "dictionary" in e.value.message
    ins, outs = CALLS[APP]
    text = text_of(APP, ins, outs).replace(
        "backend_config = {}", "backend_config = {}, has_side_effect = false, operand_layouts = [dense<[3, 2, 1, 0]> : "
        "tensor<4xindex>, dense<[3, 2, 1, 0]> : tensor<4xindex>], output_operand_aliases = "
        "[#stablehlo.output_operand_alias<output_tuple_indices = [0], operand_index = 0, operand_tuple_indices = []>]")
    assert plan(plugin, text)["steps"][0]["library"] == "paged_append"


def test_bytes_of_a_step_are_those_it_moves(plugin):
    """Of a cache's pages, the rows named; the whole pages where they are copied."""
    ins, outs = CALLS[ATT]
    big = [((1000, 2, 16, 64), "bf16") if t[0] == PAGES else t for t in ins]
    step = plan(plugin, text_of(ATT, big, outs))["steps"][0]
    assert step["algorithmic_bytes"] == 2 * 3 * 4 * 64 * 2 + 4 * 15 + 4 * 3 + 2 * 15 * 2 * 16 * 64 * 2
    step = plan(plugin, _append(True))["steps"][0]
    assert step["algorithmic_bytes"] == 4 * 7 * 2 * 64 * 2 + 4 * 7
    step = plan(plugin, _append(False))["steps"][0]
    assert step["algorithmic_bytes"] == 4 * 7 * 2 * 64 * 2 + 4 * 7 + 4 * 8 * 2 * 16 * 64 * 2


def test_refuses_shapes_whose_products_wrap(plugin):
    """2^32 x 2^32 rows are no rows in 64 bits."""
    big = ((2 ** 32, 2 ** 32, 8), "f32")
    with pytest.raises(PjrtError) as e:
        plan(plugin, text_of("pjrtx.add_rms_norm", [big, ((8,), "f32")], [big]))
    assert e.value.code == UNIMPLEMENTED and "2^60" in e.value.message
    pages = ((2 ** 32, 2 ** 32, 16, 64), "bf16")
    ins, outs = CALLS[ATT]
    with pytest.raises(PjrtError) as e:
        plan(plugin, text_of(ATT, [pages if t[0] == PAGES else t for t in ins], outs))
    assert e.value.code == UNIMPLEMENTED


def test_performance_cases_leave_room_in_the_fixed_block(plugin):
    """What a case's program holds between its steps, besides results, which lie
    in the caller's memory: within the allocation-free call's block, at the
    largest rows of 8 bits that a draw's bound lets pass too."""
    import random

    import torch

    from perf import operators as cases

    room = plugin.lib.pjrtx_noalloc_scratch_bytes()
    size = {"bf16": 2, "f16": 2, "f32": 4, "i8": 1, "i32": 4}
    rng = random.Random(5)
    most = [{"kind": "norm", "rows": r, "dim": d, "quantize": True, "dtype": t}
            for r, d, t in ((8200, 8192, "bf16"), (8192, 8256, "f16"), (16384, 4160, "bf16"), (4192, 16384, "f16"))]
    most = [c for c in most if cases.work(c)["bytes"] <= cases._MOST and cases._held(c) <= 4 * cases._MOST]
    assert len(most) == 4
    for c in most + [c for c in cases.listed() if c["kind"] == "norm"] + [cases.draw(rng) for _ in range(300)]:
        if c["kind"] != "norm":
            continue
        x = torch.empty((c["rows"], c["dim"]), dtype=cases._TORCH[c["dtype"]], device="meta")
        text = cases._program(c, [x, x, x[0]])
        line = next(s for s in text.splitlines() if s.strip().startswith(("return ", "func.return ", "stablehlo.return ")))
        results = 0
        for t in re.findall(r"tensor<([^>]*)>", line):
            *dims, name = t.split("x")
            results += size[name] * int(np.prod([int(d) for d in dims]))
        held = sum(n for s in plan(plugin, text)["steps"] for n in s["out_bytes"]) - results
        assert 0 <= held <= room, (c, held)


def test_refuses_a_scale_whose_scores_are_no_floats(plugin):
    """Scores are taken times log2(e): 3e38 of that is beyond f32, and a score
    of 0 would not be 0."""
    ins, outs = CALLS[ATT]
    for scale in (3e38, -2.5e38):
        with pytest.raises(PjrtError) as e:
            plan(plugin, text_of(ATT, ins, outs, {"scale": scale}))
        assert e.value.code == INVALID and "scale" in e.value.message
    assert plan(plugin, text_of(ATT, ins, outs, {"scale": 2.0 ** 127}))["steps"]
