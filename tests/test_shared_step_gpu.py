"""What BatchedDecoder reports and refuses where a step runs under a plan."""
import pytest
import torch

pytestmark = pytest.mark.gpu
VOCAB = 151936


def _tokens(n, seed):
    return torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _forked(weights, n=3, length=300):
    """A decoder whose sequences 0 .. n - 1 share their first positions, its plan and a step's arguments."""
    from batched import BatchedDecoder
    from paged import PrefixPlan
    bd = BatchedDecoder(weights, num_seqs=6, max_rows=64, num_layers=2, paged=True, num_pages=24)
    bd.prefill_parallel([_tokens(length, 1) + [0]], seqs=[0])
    bd.fork(0, list(range(1, n)), length)
    for s in range(n):
        bd.reserve(s, length)
    dev = dict(dtype=torch.int32, device=bd.dev)
    step = (torch.arange(n, **dev), torch.full((n,), length, **dev), torch.arange(5, 5 + n, **dev))
    return bd, PrefixPlan([n], [length], 16, 8, 128, max_length=length + 10), step


def test_status_reports_what_the_attention_recorded(weights_2l):
    bd, plan, step = _forked(weights_2l)
    want = bd.step(*step, 300, prefix=plan).clone()
    assert bd.status() == 0 and plan.status() == 0
    row = bd.page_table[0].clone()
    bd.page_table[0, 0] = -1                            # a shared page: read by the attention, not written
    bd.step(*step, 300, prefix=plan)
    assert bd.status() == 3 and bd.status() == 0
    assert plan.status() == 3 and plan.status() == 0
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        bd.step(*step, 300, prefix=plan)
    g.replay()
    assert bd.status() == 3 and plan.status() == 3
    bd.page_table[0].copy_(row)
    assert torch.equal(bd.step(*step, 300, prefix=plan), want) and bd.status() == 0 and plan.status() == 0
