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


@pytest.mark.parametrize("position", [-1, 2048, 1 << 30])
def test_positions_outside_the_cache_are_refused(weights_2l, position):
    """With a plan as without one."""
    bd, plan, step = _forked(weights_2l)
    for prefix in (None, plan):
        with pytest.raises(RuntimeError, match="outside the KV cache"):
            bd.step(*step, position, prefix=prefix)


@pytest.mark.parametrize("when", ["prompt", "suffixes", "answers"])
def test_generate_shared_raises_what_any_of_its_steps_recorded(weights_2l, monkeypatch, when):
    """A page that is missing during one step only, while the prefix, the
    suffixes or the answers are computed."""
    from batched import BatchedDecoder
    bd = BatchedDecoder(weights_2l, num_seqs=4, max_rows=64, num_layers=2, paged=True, num_pages=24)
    prefix, suffixes = _tokens(200, 2), [_tokens(4, 3), _tokens(70, 4), _tokens(9, 5)]
    want = bd.generate_shared(prefix, suffixes, 4)
    bd.release([0, 1, 2])
    plain, steps = BatchedDecoder.step, []

    def step(self, *args, **kw):
        kind = "prompt" if kw.get("prefix") is None else "suffixes" if kw["prefix"].rows != 3 else "answers"
        steps.append(kind)
        if steps.count(kind) != 1 + (kind == "prompt") or kind != when:
            return plain(self, *args, **kw)
        row = self.page_table[0].clone()
        self.page_table[0, 0] = -1
        try:
            return plain(self, *args, **kw)
        finally:
            self.page_table[0].copy_(row)

    monkeypatch.setattr(BatchedDecoder, "step", step)
    with pytest.raises(RuntimeError, match="recorded error 3"):
        bd.generate_shared(prefix, suffixes, 4)
    assert set(steps) == {"prompt", "suffixes", "answers"}
    monkeypatch.undo()
    bd.release([0, 1, 2])
    assert bd.generate_shared(prefix, suffixes, 4) == want and bd.status() == 0


@pytest.mark.parametrize("prefix,suffixes,new", [
    (300, [3, 70, 130], 20),     # a partly filled page of each; one more for the last
    (256, [0, 0, 0], 1),         # shared up to position 254: nothing shared of page 1
    (256, [1, 1, 1], 129),       # whole pages shared
    (5, [0, 300, 0], 4),
])
def test_generate_shared_takes_all_its_pages_or_none(weights_2l, prefix, suffixes, new):
    from batched import BatchedDecoder
    prompt, tails = _tokens(prefix, 6), [_tokens(n, 7 + i) for i, n in enumerate(suffixes)]
    bd = BatchedDecoder(weights_2l, num_seqs=4, max_rows=64, num_layers=2, paged=True, num_pages=24)
    want = bd.generate_shared(prompt, tails, new)
    used = bd.pages_in_use
    exact = BatchedDecoder(weights_2l, num_seqs=4, max_rows=64, num_layers=2, paged=True, num_pages=used + 1)
    exact.reserve(3, 0)
    assert exact.generate_shared(prompt, tails, new) == want and exact.pages_in_use == used + 1
    exact.release([0, 1, 2])
    exact.reserve(3, 128)                               # one page fewer
    for _ in range(2):                                  # and again: it holds none
        with pytest.raises(RuntimeError, match="exhausted"):
            exact.generate_shared(prompt, tails, new)
        assert exact.pages_in_use == 2 and exact.page_table[:3].cpu().tolist() == exact.pages.table[:3]
        assert all(page < 0 for row in exact.pages.table[:3] for page in row)
