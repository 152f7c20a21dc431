"""A plan that is dropped while calls on another stream than its own still read it."""
import pytest
import torch

from paged_helpers import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("in_step", [False, True])
def test_its_memory_is_kept(weights_2l, in_step):
    from batched import BatchedDecoder
    from paged import PrefixPlan
    side = torch.cuda.Stream()
    if in_step:
        bd = BatchedDecoder(weights_2l, num_seqs=2, num_layers=2, paged=True, num_pages=8)
        bd.prefill_parallel([list(range(301))], seqs=[0])
        bd.fork(0, [1], 300)
        for s in range(2):
            bd.reserve(s, 300)
        dev = dict(dtype=torch.int32, device=bd.dev)
        args = torch.arange(2, **dev), torch.full((2,), 300, **dev), torch.arange(2, **dev), 300
        plan = PrefixPlan([2], [300], 16, 8, 128, max_length=310)
        call = lambda p: bd.step(*args, prefix=p).clone()  # noqa: E731
    else:
        c = Case(torch.float16, 128, 2, 2, 64, [6], [640], [40, 3], seed=50)
        plan = c.plan()
        call = lambda p: c.run(p)[0]  # noqa: E731
    want = call(plan)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)                  # about 0.1 s
        got = call(plan)
    ptr, n = plan.words.data_ptr(), plan.words.numel()
    del plan
    later = [torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(8)]
    assert all(t.data_ptr() != ptr for t in later)
    assert not side.query()                             # it was still to be read
    torch.cuda.synchronize()
    assert torch.equal(got, want)
