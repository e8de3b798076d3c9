"""The kernels for beams and adapters right behind products that let their successors in early, with the switch that makes launches
programmatic on: bit for bit what they give behind products that have ended."""

import pytest
import torch

from flashdecode_cuda_b200 import kernels as K
from flashdecode_cuda_b200.parts.linear import matmul

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture
def early():
    def switch(on):
        K.set_pdl(on)
    yield switch
    K.set_pdl(False)
    K.lora_set_form(0)
    K.beam_select_set_form(0)


@pytest.mark.parametrize("T,form", [(4, 1), (16, 1), (40, 1), (128, 1), (128, 2), (300, 1), (300, 2), (100, 0)])
def test_an_adapter_behind_a_product(early, T, form):
    g = torch.Generator().manual_seed(T)
    Kd, N, R = (2048, 4096, 16) if form else (2048, 4100, 12)                   # 0: sizes for the CUDA cores
    bf = lambda *s: torch.randn(*s, generator=g).bfloat16().to(DEV)
    x, w, a, b = bf(T, Kd), bf(N, Kd) * Kd ** -0.5, bf(2, R, Kd) * Kd ** -0.5, bf(2, N, R) * R ** -0.5
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    rest = (torch.ones(2, device=DEV), i32([R, R]), i32(list(range(T))), i32([0, T // 2, T]), i32([1, 0]))
    K.lora_set_form(form)
    y = torch.empty(T, N, dtype=torch.bfloat16, device=DEV)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)

    def step(between):
        y.fill_(50.0)                                            # what a product that has not ended leaves
        matmul(x, w, None, y, status=st)
        between()
        K.lora_add(x, a, b, *rest, y, status=st)
        return y.clone()
    want = step(torch.cuda.synchronize)
    early(True)
    for _ in range(10):
        assert torch.equal(step(lambda: None), want)
    assert int(st.item()) == 0


@pytest.mark.parametrize("rows,form", [(4, 1), (4, 2), (16, 1), (64, 1), (64, 2)])
def test_a_selection_behind_the_product_of_the_logits(early, rows, form):
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, 1024, generator=g).bfloat16().to(DEV)
    w = torch.randn(20000, 1024, generator=g).bfloat16().to(DEV) * 0.05
    logits, scores = torch.empty(rows, 20000, device=DEV), torch.zeros(rows, device=DEV)
    start = torch.arange(0, rows + 1, 4, dtype=torch.int32, device=DEV)
    n = len(start) - 1
    out = [torch.empty(n, 8, device=DEV)] + [torch.empty(n, 8, dtype=torch.int32, device=DEV) for _ in range(2)]
    K.beam_select_set_form(form)

    def step(between):
        logits.fill_(50.0)
        matmul(x, w, None, logits)
        between()
        K.beam_select(logits, scores, start, *out)
        return [o.clone() for o in out]
    want = step(torch.cuda.synchronize)
    early(True)
    for _ in range(10):
        assert all(torch.equal(p, q) for p, q in zip(step(lambda: None), want))
