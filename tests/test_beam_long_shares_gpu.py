"""GPU: selections of so many rows that a wave walks 3 to 122 chunks of its row (2048
logits of 16 bits, 1024 of f32), against the definition in 64 bits on the device.

Tolerance of a beam's normaliser, for any length of a row and any values: the error of
log(sum) is at most the largest relative error of the sum's terms and of its additions.
A term's argument (x - m) log2 e is rounded once, by 2^-21 ln 2 below 16 and 2^-20 ln 2
below 32 (0.69 of 2^-20); terms beyond weigh less than 2^26 2^-32.  log2 e as an fp32
number is off by 1.4e-8 of itself, 17 x 0.69 x 1.4e-8 = 0.17 of 2^-20 for terms 2^-17
of the largest (V of them count as much as it).  The exponential: 1 ulp, 2^-23,
0.13 of 2^-20.  The additions of a chunk: at most 8 roundings of 2^-24 in a row, 0.5 of
2^-20; chunks, lanes and waves meet in fp64.  Together 1.5 of 2^-20, below 2^-19.  The
score adds its own rounding, half a step of fp32."""
import pytest
import torch

import nvjsel

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SUM = 2.0 ** -19


@pytest.mark.parametrize("b,w,v,dtype", [(32, 8, 248320, "bf16"), (33, 64, 248320, "bf16"), (33, 64, 100003, "f32"),
                                         (33, 64, 100003, "f16")])
def test_rows_of_few_values(b, w, v, dtype):
    """Rows whose sums round the same way at every step: one larger value per lane and chunk's
    worth of the first logits, the rest equal, and rows that climb by a little in every chunk."""
    n = b * w
    at = torch.arange(v, device="cuda")
    logits = torch.empty(n, v, dtype=DT[dtype], device="cuda")
    low = torch.linspace(-9.0, -0.05, n, device="cuda")
    for r in range(n):
        if r % 2:
            x = torch.where(at < 512, 0.0, low[r])
        else:
            x = (at // 1024) * (low[r].abs() / 128) - 3.0
        logits[r] = x.to(DT[dtype])
    scores = torch.zeros(b, w, device="cuda")
    got, parents, tokens = (x.cpu() for x in nvjsel.beam_search_select(logits.reshape(b, w, v), scores))
    for i in range(b):
        l = logits.reshape(b, w, v)[i].double()
        norm = l.logsumexp(1)
        for j in range(w):
            p, t = int(parents[i, j]), int(tokens[i, j])
            want = float(l[p, t] - norm[p])
            assert abs(float(got[i, j]) - want) <= SUM + 2.0 ** -24 * abs(want), (i, j, p, float(got[i, j]) - want)
