"""Bounded waits of the kernels on 8-bit rows and caches that run out: reported by a counter, and harmless.  (In a file of its own that runs last: other tests ask that no
wait has run out in the process.)"""
import pytest
import torch

from kvad_b200.ops import Ops, attention_int8_wait_timeouts, linear_int8_wait_timeouts, wait_test_hooks
from tests.test_gpu_int8 import DT, Step

pytestmark = pytest.mark.gpu


def goes_without(library, count, run, out):
    """The first copy of every block is left out: its wait runs out after the (shortened) limit, copies in flight are waited for, the launch returns without writing, and
    the next one is whole."""
    run()
    torch.cuda.synchronize()
    want, before = out.clone(), count()
    out.fill_(7)
    try:
        wait_test_hooks(library, 4096, True)
        run()
        torch.cuda.synchronize()
        assert count() > before and (out == 7).all()
    finally:
        wait_test_hooks(library)
    after = count()
    run()
    assert count() == after and torch.equal(out, want) and not (out == 7).all()


@pytest.mark.parametrize("form", [64, 128, 256, 512])
def test_weights_that_never_come(form):
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    a, w = (torch.randint(-127, 128, s, generator=g, device="cuda", dtype=torch.int8) for s in ((200, 512), (300, 512)))
    sa, sw = torch.ones(200, device="cuda"), torch.ones(300, device="cuda")
    out = torch.empty(200, 300, device="cuda")
    goes_without("linear_int8", linear_int8_wait_timeouts, lambda: Ops(torch.float32).linear_int8(a, sa, w, sw, None, out, form=form), out)


@pytest.mark.parametrize("library,dtype,new,before,hd", [("attention_int8", "bfloat16", [1, 1, 1], [63, 64, 500], 64), ("attention_int8", "float32", [1, 1], [200, 3], 128),
                                                        ("attention_int8", "float32", [70, 3], [0, 64], 32), ("attention_int8_prompt", "bfloat16", [200, 65], [0, 300], 64),
                                                        ("attention_int8_prompt", "bfloat16", [130], [77], 128)])
def test_pages_that_never_come(library, dtype, new, before, hd):
    step = Step(new, before, 2, hd)
    step.fill(5)
    q = torch.randn(step.rows, 4 * hd, device="cuda").to(DT[dtype])
    out = torch.empty_like(q)
    lens = torch.tensor(step.lens, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    goes_without(library, attention_int8_wait_timeouts,
                 lambda: Ops(DT[dtype]).attention_int8(q, out, starts, lens, len(new), max(new), step.table, *step.pages(), 4, hd ** -0.5), out)
