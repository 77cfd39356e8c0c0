"""Operators of a beam-search decode step, as data to measure: the LM head with
4-bit weights and group scales (dense logits, and greedy top-1 without logits),
the selection over beams and vocabulary, and the reordering of the beams'
states that follows it.

``own`` false: the operators' plain forms in elementary torch operations; true:
the calls of the public entry points of ``nvjsel``.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
VOCAB, HIDDEN = 248320, 1024  # the served model's LM head


def _nvjsel():
    pkg = os.path.abspath("nano-vllm-jax_amd")  # the package's folder is not importable by its own name
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import nvjsel

    return nvjsel


def _w4(name, kind, rows, vocab, hidden, group, act, zeros):
    return {"name": name, "kind": kind, "rows": rows, "vocab": vocab, "hidden": hidden, "group": group, "act": act,
            "zeros": zeros}


def _beam(name, batch, beams, vocab, k, dtype, ended=False, masked=False):
    return {"name": name, "kind": "beam", "batch": batch, "beams": beams, "vocab": vocab, "k": k, "dtype": dtype,
            "ended": ended, "masked": masked}


def _reorder(name, batch, beams, layers, heads, length, width, dtype, ragged, spare):
    return {"name": name, "kind": "reorder", "batch": batch, "beams": beams, "layers": layers, "heads": heads,
            "length": length, "width": width, "dtype": dtype, "ragged": ragged, "spare": spare}


def listed():
    return [
        # one interactive sequence, greedy, on the served model's head in 4 bits
        _w4("w4_greedy_one", "w4_greedy", 1, VOCAB, HIDDEN, 128, "bf16", False),
        # a small server's greedy step on a half-precision checkpoint with zero points, a wider hidden
        _w4("w4_greedy_rows8", "w4_greedy", 8, 151936, 2560, 64, "f16", True),
        # four requests of four beams: the logits that the selection reads
        _w4("w4_logits_rows16", "w4_logits", 16, VOCAB, HIDDEN, 128, "bf16", False),
        # a small model of an odd vocabulary with fine groups, zero points and fp32 activations
        _w4("w4_logits_f32_odd", "w4_logits", 3, 50257, 768, 32, "f32", True),
        # a full server's sampled or beam step: 64 rows of dense logits
        _w4("w4_logits_rows64", "w4_logits", 64, 128256, 2048, 128, "bf16", False),
        # the smallest call: one request, four beams, twice as many candidates as beams
        _beam("beam_one", 1, 4, 32000, 8, "bf16"),
        # a few requests on the served vocabulary
        _beam("beam_rows32", 8, 4, VOCAB, 8, "bf16"),
        # fp32 logits of an odd vocabulary with ended and unborn beams and masked tokens
        _beam("beam_f32_odd_masked", 5, 5, 50257, 10, "f32", True, True),
        # a full server: 32 requests of eight beams
        _beam("beam_rows256", 32, 8, VOCAB, 16, "bf16"),
        # one request's recurrent states: latency
        _reorder("reorder_small", 1, 4, 4, 8, 64, 64, "f32", False, 0),
        # key and value caches by heads, each request at its own length
        _reorder("reorder_caches", 16, 4, 12, 2, 2048, 128, "bf16", True, 0),
        # recurrent states of many layers in a slot table with room for other requests
        _reorder("reorder_recurrent", 16, 4, 12, 16, 128, 128, "f32", False, 16),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["w4_greedy", "w4_logits", "w4_logits", "beam", "beam", "reorder"])
    if kind == "reorder":
        batch, beams = _log_uniform(rng, 1, 16), rng.randint(2, 8)
        layers, heads = rng.randint(1, 12), rng.choice([1, 2, 3, 8, 16])
        length, width = _log_uniform(rng, 16, 2048), rng.choice([24, 64, 80, 96, 128, 256])
        dtype = rng.choice(["bf16", "f16", "f32"])
        # at most what the largest listed case moves
        while batch * beams * layers * heads * length * width * _SIZE[dtype] > 16 * 4 * 12 * 16 * 128 * 128 * 4:
            batch, layers, length = max(1, batch - 2), max(1, layers - 1), max(16, length // 2)
        return {k: v for k, v in _reorder("", batch, beams, layers, heads, length, width, dtype, rng.random() < 0.5,
                                          rng.choice([0, 3, 16])).items() if k != "name"}
    vocab = _log_uniform(rng, 2000, VOCAB)  # any size, odd ones too
    if rng.random() < 0.5:
        vocab -= vocab % 64  # a padded vocabulary
    if kind == "beam":
        beams = rng.choice([2, 3, 4, 5, 6, 8, 10, 16])
        batch = _log_uniform(rng, 1, 256 // beams)
        return {k: v for k, v in _beam("", batch, beams, vocab, rng.choice([beams, 2 * beams]),
                                       rng.choice(["bf16", "f16"] if batch * beams > 128 else ["bf16", "f16", "f32"]),
                                       rng.random() < 0.4, rng.random() < 0.3).items() if k != "name"}
    group = rng.choice([32, 64, 128, 128])
    hidden = rng.choice([512, 768, 1024, 1024, 1536, 2048, 2560, 4096]) - group * rng.choice([0, 0, 1])
    while vocab * hidden > VOCAB * HIDDEN:
        vocab //= 2
    act = rng.choice(["bf16", "bf16", "f16", "f32"])
    rows = _log_uniform(rng, 1, 32 if act == "f32" else 64)
    return {k: v for k, v in _w4("", kind, rows, vocab, hidden, group, act, rng.random() < 0.4).items() if k != "name"}


# ---------------------------------------------------------------- inputs


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _prepare_w4(c, g):
    """Weights N(0, 0.02) rounded to 4 bits by groups, and hidden rows whose
    logits spread by about 2 with a few tokens well above the bulk."""
    v, h, n, gs = c["vocab"], c["hidden"], c["rows"], c["group"]
    w = torch.empty((v, h // gs, gs), device="cuda").normal_(0.0, 0.02, generator=g)
    sdt = torch.bfloat16 if c["act"] == "bf16" else torch.float16
    if c["zeros"]:
        lo, hi = w.amin(2, keepdim=True), w.amax(2, keepdim=True)
        scales = ((hi - lo) / 15.0).to(sdt)
        zeros = torch.clamp(torch.round(-lo / scales.float()), 0, 15)
        q = torch.clamp(torch.round(w / scales.float()) + zeros, 0, 15)
    else:
        scales = (w.abs().amax(2, keepdim=True) / 7.0).to(sdt)
        zeros = None
        q = torch.clamp(torch.round(w / scales.float()), -8, 7) + 8.0
    scale = 2.0 / (0.02 * math.sqrt(h))
    x = torch.randn(n, h, device="cuda", generator=g) * scale
    for top in (20.0, 12.0, 10.0):
        t = torch.randint(0, v, (n,), device="cuda", generator=g)
        peak = top * (0.75 + 0.25 * torch.rand(n, 1, device="cuda", generator=g))
        x += peak / (h * 4e-4) * w[t].reshape(n, h)
    q = q.reshape(v, h // 2, 2).to(torch.uint8)
    s = {"qweight": (q[:, :, 0] | (q[:, :, 1] << 4)).contiguous(), "scales": scales.reshape(v, h // gs).contiguous(),
         "zeros": None if zeros is None else zeros.reshape(v, h // gs).to(torch.uint8).contiguous(),
         "hidden": x.to(_DT[c["act"]]).reshape(n, 1, h)}
    if own:  # laid out once, when the checkpoint is loaded
        s["head"] = _nvjsel().pack_lm_head_w4(s["qweight"], s["scales"], s["zeros"])
    return s


def _prepare_beam(c, g):
    """Logits with a Zipf tail; cumulative scores of beams some steps old."""
    b, w, v = c["batch"], c["beams"], c["vocab"]
    x = torch.empty(b * w, v, device="cuda").exponential_(1.0, generator=g)
    x = x * (1.05 + 0.25 * torch.rand(b * w, 1, device="cuda", generator=g))
    x = (x + torch.randn(b * w, v, device="cuda", generator=g)).reshape(b, w, v).to(_DT[c["dtype"]])
    if c["masked"]:  # a constrained step: half of the tokens at the type's lowest value, a few at -inf
        x[torch.rand(b, w, v, device="cuda", generator=g) < 0.5] = torch.finfo(x.dtype).min
        x[torch.rand(b, w, v, device="cuda", generator=g) < 0.01] = -math.inf
    scores = -torch.cumsum(0.5 * torch.rand(b, w, device="cuda", generator=g), 1) - 10.0 * torch.rand(
        b, 1, device="cuda", generator=g)
    finished = None
    if c["ended"]:
        finished = torch.rand(b, w, device="cuda", generator=g) < 0.25
        scores[:, -1] = -math.inf  # a beam that is not live yet
    return {"logits": x, "scores": scores, "k": c["k"], "finished": finished, "end": 2}


def _prepare_reorder(c, g):
    n = c["batch"] * c["beams"]
    shape = (n + c["spare"], c["heads"], c["length"], c["width"])
    states = [torch.empty(shape, dtype=_DT[c["dtype"]], device="cuda").normal_(generator=g) for _ in range(c["layers"])]
    parents = torch.randint(0, c["beams"], (c["batch"], c["beams"]), device="cuda", generator=g, dtype=torch.int32)
    slots = lengths = None
    if c["spare"]:
        slots = torch.randperm(n + c["spare"], device="cuda", generator=g)[:n].to(torch.int32)
        slots = slots.reshape(c["batch"], c["beams"])
    if c["ragged"]:
        lengths = torch.randint(1, c["length"] + 1, (c["batch"],), device="cuda", generator=g, dtype=torch.int32)
    return {"states": states, "parents": parents, "slots": slots, "lengths": lengths}


def prepare(case, seed):
    g = _gen(seed)
    s = (_prepare_beam if case["kind"] == "beam" else _prepare_reorder if case["kind"] == "reorder" else _prepare_w4)(
        case, g)
    s["kind"] = case["kind"]
    return s


# ---------------------------------------------------------------- plain forms


def _w4_logits(s):
    q, x = s["qweight"], s["hidden"].reshape(s["hidden"].shape[0], -1)
    v, groups = s["scales"].shape
    w = torch.stack((q & 15, q >> 4), 2).reshape(v, groups, -1).float()
    w = (w - (8.0 if s["zeros"] is None else s["zeros"].float()[:, :, None])) * s["scales"].float()[:, :, None]
    return x.float() @ w.reshape(v, -1).T


def _beam_select(s):
    l, scores = s["logits"].double(), s["scores"].double()
    b, w, v = l.shape
    m = l.amax(2, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    l = l - m
    total = scores[:, :, None] + (l - torch.log(torch.exp(l).sum(2, keepdim=True)))
    total = torch.where((scores == -math.inf)[:, :, None], -math.inf, total)
    if s["finished"] is not None:
        total = torch.where(s["finished"][:, :, None], -math.inf, total)
        total[:, :, s["end"]] = torch.where(s["finished"], scores, total[:, :, s["end"]])
    total = total.reshape(b, w * v)
    # the lowest place first among equal ones: a stable sort of enough of the largest, in order of place
    place = torch.topk(total, min(w * v, s["k"] + 240), dim=1).indices.sort(dim=1).values
    value, order = torch.sort(total.gather(1, place), dim=1, descending=True, stable=True)
    value, place = value[:, : s["k"]], place.gather(1, order[:, : s["k"]])
    none = value == -math.inf
    return (value.float(), torch.where(none, -1, place // v).to(torch.int32),
            torch.where(none, -1, place % v).to(torch.int32))


def _reorder_states(s):
    b, w = s["parents"].shape
    slots = torch.arange(b * w, device="cuda").reshape(b, w) if s["slots"] is None else s["slots"].long()
    to, source = slots.reshape(-1), slots.gather(1, s["parents"].long()).reshape(-1)
    if s["lengths"] is not None:
        valid = torch.arange(s["states"][0].shape[2], device="cuda") < s["lengths"].repeat_interleave(w)[:, None]
        valid = valid[:, None, :, None]
    for t in s["states"]:
        moved = t[source]
        t[to] = moved if s["lengths"] is None else torch.where(valid, moved, t[to])
    return s["states"]


def run(state):
    kind = state["kind"]
    if own:
        nvjsel = _nvjsel()
        if kind == "w4_greedy":
            return nvjsel.lm_head_greedy_top1_hip(state["hidden"], state["head"], reduce_cast=0, return_best=True)
        if kind == "w4_logits":
            return nvjsel.lm_head_logits_hip(state["hidden"], state["head"])
        if kind == "beam":
            return nvjsel.beam_search_select(state["logits"], state["scores"], num_candidates=state["k"],
                                             finished=state["finished"], end_token=state["end"])
        nvjsel.reorder_beam_states(state["states"], state["parents"], slots=state["slots"], lengths=state["lengths"],
                                   length_dim=None if state["lengths"] is None else 2)
        return state["states"]
    if kind == "w4_greedy":
        best = torch.max(_w4_logits(state), dim=1)  # compared as they are: fp32
        return best.indices[:, None].to(torch.int32), best.values
    if kind == "w4_logits":
        return _w4_logits(state).to(state["hidden"].dtype)
    return _beam_select(state) if kind == "beam" else _reorder_states(state)


# ---------------------------------------------------------------- work and 64-bit results


def work(case):
    if case["kind"] == "beam":
        # logits once, K scores, parents and tokens; a subtraction, an exponential, a sum and a comparison per value
        n, b = case["batch"] * case["beams"] * case["vocab"], case["batch"]
        return {"bytes": n * _SIZE[case["dtype"]] + b * (case["k"] * 12 + case["beams"] * 5), "flops": 4 * n}
    if case["kind"] == "reorder":
        # random parents: a beam moves unless it is its own parent; a source is read if another beam takes it
        w = case["beams"]
        row = case["heads"] * case["length"] * case["width"] * _SIZE[case["dtype"]] * (0.5 if case["ragged"] else 1.0)
        beams = (1 - 1 / w) + (1 - (1 - 1 / w) ** (w - 1))
        return {"bytes": case["layers"] * case["batch"] * w * row * beams, "flops": 0}
    v, h, n = case["vocab"], case["hidden"], case["rows"]
    out = n * v * _SIZE[case["act"]] if case["kind"] == "w4_logits" else n * 8
    groups = v * (h // case["group"]) * (3 if case["zeros"] else 2)
    return {"bytes": v * h // 2 + groups + n * h * _SIZE[case["act"]] + out, "flops": 2 * n * v * h}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "reorder":
        parents = s["parents"].tolist()
        slots = s["slots"].tolist() if s["slots"] is not None else [
            [b * case["beams"] + w for w in range(case["beams"])] for b in range(case["batch"])]
        lengths = s["lengths"].tolist() if s["lengths"] is not None else [case["length"]] * case["batch"]
        result = []
        for t in s["states"]:
            new = t.clone()
            for b in range(case["batch"]):
                for w in range(case["beams"]):
                    new[slots[b][w], :, : lengths[b]] = t[slots[b][parents[b][w]], :, : lengths[b]]
            result.append(new)
        return result
    if case["kind"] == "beam":
        values = []
        for b in range(case["batch"]):
            of = []
            for w in range(case["beams"]):
                score = s["scores"][b, w].double()
                if s["finished"] is not None and bool(s["finished"][b, w]):
                    of.append(score.reshape(1))
                elif bool(torch.isfinite(score)):
                    of.append(score + torch.log_softmax(s["logits"][b, w].double(), 0))
            of = torch.sort(torch.cat(of + [torch.full((case["k"],), -math.inf, dtype=torch.float64, device="cuda")]),
                            descending=True).values
            values.append(of[: case["k"]])
        return [torch.stack(values), None, None]
    x = s["hidden"].double().reshape(case["rows"], case["hidden"])
    parts = []
    for v0 in range(0, case["vocab"], 16384):  # even and odd places of a row apart
        q = s["qweight"][v0:v0 + 16384]
        scale = s["scales"][v0:v0 + 16384].double().repeat_interleave(case["group"] // 2, 1)
        zero = 8.0 if s["zeros"] is None else s["zeros"][v0:v0 + 16384].double().repeat_interleave(
            case["group"] // 2, 1)
        even, odd = ((q % 16).double() - zero) * scale, (torch.div(q, 16, rounding_mode="floor").double() - zero) * scale
        parts.append(x[:, 0::2].contiguous() @ even.T.contiguous() + x[:, 1::2].contiguous() @ odd.T.contiguous())
    logits = torch.cat(parts, 1)
    return logits if case["kind"] == "w4_logits" else [None, logits.amax(1)]
