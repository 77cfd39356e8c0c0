"""Operators that answer for tokens, as data to measure: log probabilities of
given tokens with entropy and top alternatives (over logits, with their
gradient, and from the hidden states without logits), and low-rank adapters of
many requests beside a shared projection.

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


_package = None


def _nvjsel():
    global _package
    if _package is None:  # looked up once, not at every call
        pkg = os.path.abspath("nano-vllm-jax_amd")  # the package's folder is not importable by its own name
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import nvjsel as _package
    return _package


def _logprobs(name, rows, vocab, top, entropy, dtype, masked=False, grad=False, padded=False):
    return {"name": name, "kind": "logprobs", "rows": rows, "vocab": vocab, "top": top, "entropy": entropy,
            "dtype": dtype, "masked": masked, "grad": grad, "padded": padded}


def _score(name, rows, vocab, hidden, act, weight, entropy, padded=False):
    return {"name": name, "kind": "score", "rows": rows, "vocab": vocab, "hidden": hidden, "act": act,
            "weight": weight, "entropy": entropy, "padded": padded}


def _adapters(name, rows, hidden, width, rank, count, act, table, prompts=False):
    return {"name": name, "kind": "adapters", "rows": rows, "hidden": hidden, "width": width, "rank": rank,
            "count": count, "act": act, "table": table, "prompts": prompts}


def listed():
    return [
        # one interactive sequence: the chosen token's log probability and 20 alternatives
        _logprobs("logprobs_one", 1, VOCAB, 20, False, "bf16"),
        # a full server's step, every row with alternatives and entropy
        _logprobs("logprobs_rows64", 64, VOCAB, 20, True, "bf16"),
        # a constrained step of a small server: fp32 logits of an odd vocabulary, masks, one row with nothing left
        _logprobs("logprobs_f32_odd_masked", 5, 50257, 5, True, "f32", masked=True),
        # the logits of a prompt's chunk, no alternatives, rows behind the last sequence
        _logprobs("logprobs_prompt", 1000, 151936, 0, True, "bf16", padded=True),
        # a policy's training step: log probabilities, entropies and the gradient of both
        _logprobs("logprobs_grad", 512, 151936, 0, True, "bf16", grad=True),
        # a small training step of fp32 logits with ignored rows and an odd vocabulary
        _logprobs("logprobs_grad_f32_odd", 37, 50257, 0, False, "f32", grad=True, padded=True),
        # prompts of 2048 tokens scored from their hidden states
        _score("score_prompt", 2048, VOCAB, HIDDEN, "bf16", "bf16", True),
        # a verifier's draft of a few tokens scored
        _score("score_draft", 24, VOCAB, HIDDEN, "bf16", "bf16", False),
        # fp32 activations, a ragged prompt, an odd vocabulary of a small model
        _score("score_f32_odd", 300, 50257, 768, "f32", "bf16", True, padded=True),
        # one token of one request at a projection of a layer's size: latency
        _adapters("adapters_one", 1, 2048, 2048, 16, 4, "bf16", "bf16"),
        # a full server's decode step at the LM head, 64 requests of 16 adapters
        _adapters("adapters_head_rows64", 64, HIDDEN, VOCAB, 16, 16, "bf16", "bf16"),
        # prompts of several requests at a projection of a layer's size, fp16, rank 64
        _adapters("adapters_prompt", 2000, 2560, 4096, 64, 6, "f16", "f16", prompts=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["logprobs", "logprobs", "grad", "score", "score", "adapters", "adapters"])
    if kind == "adapters":
        act = rng.choice(["bf16", "bf16", "f16", "f32"])
        table = act if act != "f32" else rng.choice(["bf16", "f16"])
        prompts = rng.random() < 0.35
        hidden = rng.choice([512, 768, 1000, 1024, 2048, 2560, 4096])
        width = _log_uniform(rng, 256, 8192) if prompts or rng.random() < 0.6 else _log_uniform(rng, 8192, VOCAB)
        rows = _log_uniform(rng, 64, 2048) if prompts else _log_uniform(rng, 1, 128)
        case = _adapters("", rows, hidden, width, rng.choice([4, 8, 16, 16, 24, 32, 64, 128]), rng.randint(1, 24), act,
                         table, prompts)
    else:
        vocab = _log_uniform(rng, 2000, VOCAB)  # any size, odd ones too
        if rng.random() < 0.5:
            vocab -= vocab % 64  # a padded vocabulary
        entropy, padded = rng.random() < 0.6, rng.random() < 0.3
        if kind == "score":
            act = rng.choice(["bf16", "bf16", "f16", "f32"])
            weight = act if act != "f32" else "bf16"
            hidden = rng.choice([512, 768, 1024, 1024, 1536, 2048, 2560, 4096])
            rows = _log_uniform(rng, 1, 512 if act == "f32" else 2048)
            while rows * vocab * hidden > 2048 * VOCAB * HIDDEN // (4 if act == "f32" else 1):
                rows = max(1, rows // 2)
            case = _score("", rows, vocab, hidden, act, weight, entropy, padded)
        else:
            dtype, grad = rng.choice(["bf16", "f16", "f32"]), kind == "grad"
            rows = _log_uniform(rng, 1, 512)
            while rows * vocab * _SIZE[dtype] > 512 * 151936 * 2:
                rows = max(1, rows // 2)
            case = _logprobs("", rows, vocab, 0 if grad else rng.choice([0, 1, 5, 10, 20, 32]), entropy, dtype,
                             rng.random() < 0.3, grad, padded)
    return {k: v for k, v in case.items() if k != "name"}


# ---------------------------------------------------------------- inputs


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _tokens(c, g, likely=None):
    """Half of the tokens likely ones, the others any; -1 in the rows behind the last sequence."""
    n, v = c["rows"], c["vocab"]
    t = torch.randint(0, v, (n,), device="cuda", generator=g)
    if likely is not None:
        t = torch.where(torch.rand(n, device="cuda", generator=g) < 0.5, likely, t)
    if c["padded"]:
        t[n - n // 8 - 1:] = -1
    return t


def _prepare_logprobs(c, g):
    """Logits with a Zipf tail, as an LM head gives them."""
    n, v = c["rows"], c["vocab"]
    x = torch.empty(n, v, device="cuda").exponential_(1.0, generator=g)
    x = x * (1.05 + 0.25 * torch.rand(n, 1, device="cuda", generator=g))
    x = (x + torch.randn(n, v, device="cuda", generator=g)).to(_DT[c["dtype"]])
    if c["masked"]:  # a constrained step: half of the tokens at the type's lowest value, a few at -inf
        x[torch.rand(n, v, device="cuda", generator=g) < 0.5] = torch.finfo(x.dtype).min
        x[torch.rand(n, v, device="cuda", generator=g) < 0.01] = -math.inf
    tokens = _tokens(c, g, x.argmax(1))
    if c["masked"]:  # chosen among what is allowed; and a constraint that leaves nothing
        allowed = x.topk(8, dim=1).indices.gather(1, torch.randint(0, 8, (n, 1), device="cuda", generator=g))[:, 0]
        tokens = torch.where(tokens >= 0, allowed, tokens)
        if n > 1:
            x[n // 2] = -math.inf
    s = {"logits": x, "tokens": tokens.to(torch.int32), "top": c["top"], "entropy": c["entropy"], "grad": c["grad"]}
    if c["grad"]:  # a policy's advantages over the rows, and the weight of the entropy
        s["tokens"] = tokens
        s["grad_logprobs"] = torch.randn(n, device="cuda", generator=g) / n
        s["grad_entropy"] = torch.full((n,), -0.01 / n, device="cuda") if c["entropy"] else None
    return s


def _prepare_score(c, g):
    """A tied table N(0, 0.02) and hidden rows whose logits spread by about 2,
    each with its next token and a few others above the bulk."""
    v, h, n = c["vocab"], c["hidden"], c["rows"]
    w = torch.empty((v, h), dtype=_DT[c["weight"]], device="cuda").normal_(0.0, 0.02, generator=g)
    x = torch.randn(n, h, device="cuda", generator=g) * (2.0 / (0.02 * math.sqrt(h)))
    for top in (14.0, 12.0, 10.0):
        t = torch.randint(0, v, (n,), device="cuda", generator=g)
        x += top * (0.5 + torch.rand(n, 1, device="cuda", generator=g)) / (h * 4e-4) * w[t].float()
    return {"hidden": x.to(_DT[c["act"]]), "weight": w, "tokens": _tokens(c, g, t).to(torch.int32),
            "entropy": c["entropy"]}


def _prepare_adapters(c, g):
    """Adapters whose updates are about a tenth of the projection's output; one row in eight without one."""
    n, h, d, r, k = c["rows"], c["hidden"], c["width"], c["rank"], c["count"]
    dt = _DT[c["table"]]
    a = torch.empty((k, r, h), dtype=dt, device="cuda").normal_(0.0, 1.0 / math.sqrt(h), generator=g)
    b = torch.empty((k, d, r), dtype=dt, device="cuda").normal_(0.0, 0.1 / math.sqrt(r), generator=g)
    scales = 0.5 + 1.5 * torch.rand(k, device="cuda", generator=g)
    if c["prompts"]:  # runs of rows, one request each
        runs = max(1, min(n, c["count"] + 2))
        ends = torch.randint(0, n, (runs - 1,), device="cuda", generator=g).sort().values
        of = torch.searchsorted(ends, torch.arange(n, device="cuda"), right=True)
        ids = torch.randint(0, k, (runs,), device="cuda", generator=g)[of]
    else:
        ids = torch.randint(0, k, (n,), device="cuda", generator=g)
        ids[torch.rand(n, device="cuda", generator=g) < 0.125] = -1
    s = {"x": torch.randn(n, h, device="cuda", generator=g).to(_DT[c["act"]]),
         "base": torch.randn(n, d, device="cuda", generator=g).to(_DT[c["act"]]), "a": a, "b": b, "scales": scales,
         "ids": ids.to(torch.int32)}
    if own:  # laid out once, when the adapters are loaded
        s["table"] = _nvjsel().pack_adapters(a, b, scales)
    return s


def prepare(case, seed):
    g = _gen(seed)
    s = {"logprobs": _prepare_logprobs, "score": _prepare_score, "adapters": _prepare_adapters}[case["kind"]](case, g)
    s["kind"] = case["kind"]
    return s


# ---------------------------------------------------------------- plain forms


def _row_sums(l):
    """Differences from the row's maximum (0 where nothing is left), log of their exponentials' sum, and whether
    something is left.  Sums of up to a quarter million terms are taken in 64 bits."""
    m = l.amax(1, keepdim=True)
    left = m != -math.inf
    d = l - torch.where(left, m, 0.0)
    return d, torch.log(torch.exp(d).sum(1, keepdim=True, dtype=torch.float64)).float(), left


def _plain_logprobs(l, tokens, top, entropy):
    """As the entry points return it; and the rows' log probabilities, with the entropy."""
    d, log_sum, left = _row_sums(l)
    logp = torch.where(left, d - log_sum, -math.inf)
    asked = (tokens >= 0) & (tokens < l.shape[1])
    own_logp = logp.gather(1, tokens.long().clamp(0, l.shape[1] - 1)[:, None])[:, 0]
    out = [torch.where(asked, own_logp, 0.0)]
    h = None
    if entropy:
        h = -torch.where(logp == -math.inf, 0.0, torch.exp(logp) * logp).sum(1, dtype=torch.float64).float()
        out.append(h)
    if top:
        # the lowest token first among equal ones: a stable sort of enough of the largest, in order of token
        v = l.shape[1]
        place = torch.topk(l, min(v, top + 480), dim=1).indices.sort(dim=1).values
        value, order = torch.sort(l.gather(1, place), dim=1, descending=True, stable=True)
        place = place.gather(1, order)[:, :top]
        none = value[:, :top] == -math.inf
        out += [torch.where(none, -math.inf, logp.gather(1, place)), torch.where(none, -1, place).to(torch.int32)]
    return out, logp, h


def _plain_logits(s):
    out, logp, h = _plain_logprobs(s["logits"].float(), s["tokens"], s["top"], s["entropy"])
    if not s["grad"]:
        return out
    p = torch.exp(logp)
    asked = (s["tokens"] >= 0) & (s["tokens"] < p.shape[1])
    g = torch.where(asked, s["grad_logprobs"], 0.0)[:, None]
    d = -g * p
    if h is not None:
        d -= s["grad_entropy"][:, None] * torch.where(p == 0.0, 0.0, p * (logp + h[:, None]))
    d.scatter_add_(1, s["tokens"].clamp(min=0)[:, None], g)
    some = (logp.amax(1, keepdim=True) != -math.inf)
    return out + [torch.where(some, d, 0.0).to(s["logits"].dtype)]


def _plain_adapters(s):
    out = s["base"].to(torch.float32, copy=True)  # fp32 base is not to be changed
    x = s["x"].float()
    for k in range(s["a"].shape[0]):
        of = (s["ids"] == k)[:, None]
        delta = torch.where(of, x, 0.0) @ s["a"][k].float().T
        out += s["scales"][k] * (delta @ s["b"][k].float().T)
    return out.to(s["base"].dtype)


def run(state):
    kind = state["kind"]
    if own:
        nvjsel = _nvjsel()
        if kind == "adapters":
            return nvjsel.apply_adapters(state["x"], state["base"], state["table"], state["ids"])
        if kind == "score":
            r = nvjsel.lm_head_token_logprobs(state["hidden"], state["weight"], state["tokens"], weight_layout="vh",
                                              entropy=state["entropy"], reduce_cast=0)
        elif state["grad"]:
            logits = state["logits"].detach().requires_grad_()
            r = nvjsel.token_logprobs(logits, state["tokens"], entropy=state["entropy"])
            outs = [r.logprobs] + ([r.entropy] if state["entropy"] else [])
            grads = [state["grad_logprobs"]] + ([state["grad_entropy"]] if state["entropy"] else [])
            return [t.detach() for t in outs] + list(torch.autograd.grad(outs, logits, grads))
        else:
            r = nvjsel.token_logprobs(state["logits"], state["tokens"], num_top=state["top"], entropy=state["entropy"])
        return [t for t in r if t is not None]
    if kind == "adapters":
        return _plain_adapters(state)
    if kind == "score":
        return _plain_logprobs(state["hidden"].float() @ state["weight"].float().T, state["tokens"], 0,
                               state["entropy"])[0]
    return _plain_logits(state)


# ---------------------------------------------------------------- work and 64-bit results


def work(case):
    n = case["rows"]
    if case["kind"] == "adapters":
        h, d, r, e = case["hidden"], case["width"], case["rank"], _SIZE[case["act"]]
        asked = case["count"] * (1 - (1 - 1 / case["count"]) ** n)  # adapters that some row names
        if case["prompts"]:
            asked = min(asked, case["count"] * (1 - (1 - 1 / case["count"]) ** (case["count"] + 2)))
        return {"bytes": n * (h + 2 * d) * e + asked * r * (h + d) * 2 + n * 4,
                "flops": 2 * n * r * (h + d) * (1.0 if case["prompts"] else 0.875)}
    v = case["vocab"]
    if case["kind"] == "score":
        h = case["hidden"]
        return {"bytes": v * h * _SIZE[case["weight"]] + n * (h * _SIZE[case["act"]] + 12), "flops": 2 * n * v * h}
    # a difference, an exponential, a sum and a comparison per logit; the gradient needs the whole row's sum first
    e = n * v * _SIZE[case["dtype"]]
    return {"bytes": (3 if case["grad"] else 1) * e + n * (12 + 8 * case["top"]), "flops": (8 if case["grad"] else 4) * n * v}


def _exact_rows(l, tokens, top, entropy, grads=None):
    """Row by row, from the definition, in 64 bits; laid out as ``run``'s outputs."""
    lps, ents, tops, ds = [], [], [], []
    for i, t in enumerate(tokens.tolist()):
        row = l[i].double()
        left = row[row > -math.inf]
        inside = 0 <= t < row.numel()
        if left.numel() == 0:
            lps.append(-math.inf if inside else 0.0)
            ents.append(row.new_zeros(()))
            tops.append(row.new_full((top,), -math.inf))
            ds.append(torch.zeros_like(row))
            continue
        lse = torch.logsumexp(left, 0)
        lps.append((row[t] - lse) if inside else 0.0)
        ent = lse - (torch.softmax(left, 0) * left).sum()
        ents.append(ent)
        if top:
            best = torch.sort(left, descending=True).values[:top] - lse
            tops.append(torch.cat([best, row.new_full((top - best.numel(),), -math.inf)]))
        if grads is not None:
            p = torch.softmax(row, 0)
            lp = torch.where(row > -math.inf, row - lse, 0.0)
            d = torch.zeros_like(row)
            if inside:
                d -= grads[0][i].double() * p
                d[t] += grads[0][i].double()
            if grads[1] is not None:
                d -= grads[1][i].double() * p * (lp + ent)
            ds.append(d)
    out = [torch.stack([torch.as_tensor(x, dtype=torch.float64, device=l.device) for x in lps])]
    if entropy:
        out.append(torch.stack(ents))
    if top:
        out += [torch.stack(tops), None]
    if grads is not None:
        out.append(torch.stack(ds))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logprobs":
        return _exact_rows(s["logits"], s["tokens"], s["top"], s["entropy"],
                           (s["grad_logprobs"], s["grad_entropy"]) if s["grad"] else None)
    if case["kind"] == "score":
        w = s["weight"].double().T.contiguous()
        parts = [_exact_rows(s["hidden"][i:i + 256].double() @ w, s["tokens"][i:i + 256], 0, s["entropy"])
                 for i in range(0, case["rows"], 256)]
        return [torch.cat([p[j] for p in parts]) for j in range(len(parts[0]))]
    out = s["base"].double()
    for i, k in enumerate(s["ids"].tolist()):
        if k >= 0:
            y = (s["a"][k].double() * s["x"][i].double()).sum(1)
            out[i] += s["scales"][k].double() * (s["b"][k].double() * y).sum(1)
    return out
