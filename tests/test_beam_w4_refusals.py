"""What the 4-bit LM head, the beam selection and the state reordering refuse, by
the Python entry points and by the C ABI, before any launch."""
import pytest
import torch

import nvjsel
from nvjsel import _lib

DUMMY = 0x1000  # never dereferenced: validation fails first


def head(vocab=64, hidden=128, group=32):
    return nvjsel.W4Weight(torch.zeros(1, dtype=torch.uint8), vocab, hidden, group, torch.bfloat16, False)


@pytest.mark.parametrize("kw,match", [
    ({"qweight": torch.zeros(8, 64)}, "uint8"),
    ({"qweight": torch.zeros(8, 0, dtype=torch.uint8)}, "non-empty"),
    ({"scales": torch.zeros(7, 1, dtype=torch.bfloat16)}, "scales must be"),
    ({"scales": torch.zeros(8, 1)}, "bfloat16 or float16"),
    ({"scales": torch.zeros(8, 8, dtype=torch.bfloat16)}, "group size"),
    ({"scales": torch.zeros(8, 3, dtype=torch.bfloat16)}, "scales must be"),
    ({"zeros": torch.zeros(8, 2, dtype=torch.uint8)}, "zeros must be"),
    ({"zeros": torch.zeros(8, 1)}, "zeros must be"),
    ({}, "device tensors"),
])
def test_pack_refusals(kw, match):
    args = {"qweight": torch.zeros(8, 64, dtype=torch.uint8), "scales": torch.zeros(8, 1, dtype=torch.bfloat16), **kw}
    with pytest.raises(ValueError, match=match):
        nvjsel.pack_lm_head_w4(**args)


@pytest.mark.parametrize("weight,kw,match", [
    (torch.zeros(8), {}, "must be"), (torch.zeros(128, 0), {}, "non-empty"),
    (torch.zeros(128, 8, dtype=torch.int8), {}, "dtype"), (torch.zeros(100, 8), {}, "multiple"),
    (torch.zeros(128, 8), {"group_size": 16}, "group size"),
    (torch.zeros(128, 8), {"scale_dtype": torch.float32}, "scale dtype"),
    (torch.zeros(128, 8), {"weight_layout": "x"}, "weight_layout"), (torch.zeros(128, 8), {}, "device tensors"),
])
def test_quantize_refusals(weight, kw, match):
    with pytest.raises(ValueError, match=match):
        nvjsel.quantize_lm_head_w4(weight, **kw)


@pytest.mark.parametrize("fn", [nvjsel.lm_head_logits_hip, nvjsel.lm_head_greedy_top1_hip])
def test_product_refusals(fn):
    with pytest.raises(ValueError, match="must match"):
        fn(torch.zeros(2, 1, 64), head())
    with pytest.raises(ValueError, match="non-empty"):
        fn(torch.zeros(0, 1, 128), head())
    with pytest.raises(ValueError, match="dtype"):
        fn(torch.zeros(2, 1, 128, dtype=torch.int8), head())
    with pytest.raises(ValueError, match="weight_layout"):
        fn(torch.zeros(2, 1, 128), head(), weight_layout="vh")
    with pytest.raises(ValueError, match="reduce_cast"):
        fn(torch.zeros(2, 1, 128), head(), reduce_cast=3)
    with pytest.raises(ValueError, match=r"\[B, 1, H\]"):
        fn(torch.zeros(2, 2, 128), head())
    with pytest.raises(ValueError, match="device tensors"):
        fn(torch.zeros(2, 1, 128), head())


@pytest.mark.parametrize("kw,match", [
    ({"logits": torch.zeros(2, 9)}, r"\[B, W, V\]"), ({"logits": torch.zeros(2, 3, 0)}, "non-empty"),
    ({"logits": torch.zeros(2, 3, 9, dtype=torch.int32)}, "dtype"),
    ({"logits": torch.zeros(2, 65, 9), "scores": torch.zeros(2, 65)}, r"1\.\.64"),
    ({"num_candidates": 65}, r"1\.\.64"), ({"num_candidates": 0}, r"1\.\.64"),
    ({"scores": torch.zeros(2, 4)}, "scores"), ({"scores": torch.zeros(2, 3).double()}, "scores"),
    ({"finished": torch.zeros(2, 3)}, "finished"), ({"finished": torch.zeros(2, 2, dtype=torch.bool)}, "finished"),
    ({"finished": torch.zeros(2, 3, dtype=torch.bool)}, "end_token"),
    ({"finished": torch.zeros(2, 3, dtype=torch.bool), "end_token": 9}, "end_token"),
    ({}, "device tensors"),
])
def test_select_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        nvjsel.beam_search_select(**{"logits": torch.zeros(2, 3, 9), "scores": torch.zeros(2, 3), **kw})


P = torch.zeros(2, 3, dtype=torch.int32)


@pytest.mark.parametrize("kw,match", [
    ({"parents": P.long()}, "parents"), ({"parents": P[0]}, "parents"), ({"parents": P[:0]}, "parents"),
    ({"parents": torch.zeros(1, 65, dtype=torch.int32)}, "64 beams"),
    ({"slots": P.long()}, "slots"), ({"slots": P[:1]}, "slots"),
    ({"lengths": torch.zeros(2, dtype=torch.int32)}, "go together"), ({"length_dim": 1}, "go together"),
    ({"lengths": torch.zeros(3, dtype=torch.int32), "length_dim": 1}, "lengths"),
    ({"states": []}, "states"), ({}, "device tensors"),
])
def test_reorder_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        nvjsel.reorder_beam_states(**{"states": torch.zeros(6, 4), "parents": P, **kw})


@pytest.mark.gpu
@pytest.mark.parametrize("state,kw,match", [
    (torch.zeros(5, 4), {}, "one row per beam"), (torch.zeros(()), {}, "one row per beam"),
    (torch.zeros(6, 0), {}, "empty"), (torch.zeros(6, 4, 4).transpose(1, 2), {}, "contiguous"),
    (torch.zeros(1, 4).expand(6, 4), {}, "overlap"), (torch.zeros(6, 8)[:, ::2], {}, "contiguous"),
    (torch.zeros(6, 4), {"length_dim": 0}, "length_dim"), (torch.zeros(6, 4), {"length_dim": 2}, "length_dim"),
])
def test_reorder_state_refusals(state, kw, match):
    if kw:
        kw = {**kw, "lengths": torch.zeros(2, dtype=torch.int32, device="cuda")}
    with pytest.raises(ValueError, match=match):
        nvjsel.reorder_beam_states(_on_gpu(state), P.cuda(), **kw)


def _on_gpu(t):
    """The same sizes and strides on the device."""
    base = torch.zeros(max(1, t.untyped_storage().nbytes() // t.element_size()), device="cuda")
    return base.as_strided(t.shape, t.stride())


def test_step_refusal():
    with pytest.raises(ValueError, match=r"\[B, W, H\]"):
        nvjsel.lm_head_beam_search_step(torch.zeros(2, 128), head(), torch.zeros(1, 2))


def _w4(**kw):
    a = dict(hidden=DUMMY, hd=1, packed=DUMMY, nbytes=1 << 30, sd=1, zeros=0, group=32, batch=1, H=128, V=64, rc=0, **{})
    a.update(kw)
    return [a[k] for k in ("hidden", "hd", "packed", "nbytes", "sd", "zeros", "group", "batch", "H", "V", "rc")]


@pytest.mark.parametrize("kw,code", [
    ({"hidden": None}, -1), ({"hd": 5}, -1), ({"sd": 0}, -1), ({"group": 48}, -1), ({"H": 100}, -1), ({"H": 0}, -1),
    ({"V": 0}, -1), ({"batch": 0}, -1), ({"rc": 3}, -1), ({"nbytes": 64 * 64}, -1), ({"packed": DUMMY + 8}, -1),
    ({"packed": None}, -1),
])
def test_c_products(kw, code):
    lib = _lib.load()
    assert lib.nvjsel_lm_head_w4_top1(*_w4(**kw), DUMMY, None, DUMMY, 1 << 20, None) == code and lib.nvjsel_last_error()
    assert lib.nvjsel_lm_head_w4_logits(*_w4(**kw), DUMMY, 0, 64, None) == code


def test_c_entries():
    lib = _lib.load()
    assert lib.nvjsel_lm_head_w4_top1(*_w4(), DUMMY, None, DUMMY, 8, None) == -3
    assert lib.nvjsel_lm_head_w4_top1(*_w4(), None, None, DUMMY, 1 << 20, None) == -1
    assert lib.nvjsel_lm_head_w4_logits(*_w4(), DUMMY, 0, 63, None) == -1  # rows closer than the vocabulary
    assert lib.nvjsel_lm_head_w4_logits(*_w4(), DUMMY, 4, 64, None) == -1
    assert lib.nvjsel_w4_packed_size(64, 100, 32, 0) == 0
    size = lib.nvjsel_w4_packed_size(17, 160, 32, 1)  # 2 x 2 blocks, 4 groups each
    assert size == 4 * 1024 + 512 + 256
    assert lib.nvjsel_w4_pack(DUMMY, DUMMY, DUMMY, 17, 160, 32, DUMMY, size - 1, None) == -1
    assert lib.nvjsel_w4_pack(DUMMY, None, None, 17, 160, 32, DUMMY, size, None) == -1
    assert lib.nvjsel_w4_quantize(DUMMY, 0, 0, 1, 17, 160, 32, 1, DUMMY, DUMMY, None, None) == -1
    assert lib.nvjsel_w4_quantize(DUMMY, 0, 160, 1, 17, 160, 32, 0, DUMMY, DUMMY, None, None) == -1

    need = lib.nvjsel_beam_select_workspace_size(1, 2, 4, 5000, 8)
    assert need > 0 and lib.nvjsel_beam_select_workspace_size(1, 2, 65, 5000, 8) == 0

    def select(**kw):
        a = dict(logits=DUMMY, dt=1, batch=2, beams=4, vocab=5000, bs=20000, ws_=5000, scores=DUMMY, fin=None, end=0,
                 k=8, o1=DUMMY, o2=DUMMY, o3=DUMMY, ws=DUMMY, nbytes=need, stream=None)
        a.update(kw)
        return lib.nvjsel_beam_select(*a.values())

    for kw, code in (({"logits": None}, -1), ({"dt": 3}, -1), ({"beams": 65}, -1), ({"k": 0}, -1), ({"k": 65}, -1),
                     ({"vocab": 0}, -1), ({"vocab": (1 << 26) + 1}, -1), ({"batch": 1 << 23}, -1),
                     ({"scores": None}, -1), ({"o2": None}, -1), ({"logits": DUMMY + 1}, -1), ({"bs": -1}, -1),
                     ({"fin": DUMMY, "end": 5000}, -1), ({"fin": DUMMY, "end": -1}, -1), ({"ws": None}, -3),
                     ({"nbytes": need - 1}, -3), ({"ws": DUMMY + 4}, -3)):
        assert select(**kw) == code, kw

    def reorder(count=1, parents=DUMMY, stride=4, batch=2, beams=4, slots=None, **kw):
        t = {"data": DUMMY, "row_bytes": 64, "length": 4, "token_bytes": 8, "outer": 2, "rows": 8, **kw}
        table = _lib.states([x or 0 for x in t.values()])
        return lib.nvjsel_reorder_states(table, count, parents, stride, slots, None, batch, beams, None)

    for kw in ({"count": 0}, {"parents": None}, {"stride": -1}, {"batch": 0}, {"batch": 65536}, {"beams": 65},
               {"data": None}, {"row_bytes": 63}, {"length": 0}, {"outer": 0}, {"token_bytes": 0}, {"rows": 7},
               {"length": 1 << 62}, {"length": 1 << 36, "row_bytes": 1 << 40}):  # more than 64 GB a row
        assert reorder(**kw) == -1, kw
