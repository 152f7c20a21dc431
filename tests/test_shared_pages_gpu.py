"""Sequences that share pages in the batched decoder (batched.py: fork,
reserve, release, compact, generate_shared, step(prefix=...)) against the same
sequences decoded without sharing.

The shared-prefix attention sums in another order than the split attention and
rounds its weights to fp16, so final-normed hidden states are compared through
the logits (within the batched path's tolerance) and tokens where the logits'
margin exceeds it; what only moves pages is compared bit for bit."""
import pytest
import torch

from decode_helpers import LOGIT_ATOL, MARGIN, logits_from_norm

pytestmark = pytest.mark.gpu
VOCAB = 151936


def _tokens(n, seed):
    return torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _decoder(weights, **kw):
    from batched import BatchedDecoder
    kw = {**dict(num_seqs=6, max_rows=64, num_layers=2, paged=True, num_pages=24), **kw}
    return BatchedDecoder(weights, **kw)


def _step(bd, seqs, positions, tokens, prefix=None):
    dev = dict(dtype=torch.int32, device=bd.dev)
    norm = torch.empty(len(seqs), 1024, dtype=torch.float32, device=bd.dev)
    out = bd.step(torch.tensor(seqs, **dev), torch.tensor(positions, **dev), torch.tensor(tokens, **dev),
                  max(positions), norm_out=norm, out=torch.empty(len(seqs), **dev), prefix=prefix)
    return out.cpu().tolist(), norm.cpu()


def _close(weights, got, ref):
    emb = weights["embed_weight"].cuda()
    for (t, n), (u, m) in zip(got, ref):
        for i in range(len(t)):
            a, b = logits_from_norm(n[i], emb), logits_from_norm(m[i], emb)
            assert float((a - b).abs().max()) <= LOGIT_ATOL
            top = torch.topk(b, 2).values
            if float(top[0] - top[1]) > MARGIN:
                assert t[i] == u[i]


def _run(bd, prompts, steps, prefix=None):
    """Greedy steps teacher-forced with fixed tokens, so that runs stay comparable."""
    got = []
    for s in range(steps):
        seqs, pos = list(range(len(prompts))), [len(p) - 1 + s for p in prompts]
        for i, q in zip(seqs, pos):
            bd.reserve(i, q)
        got.append(_step(bd, seqs, pos, [(p[-1] + 7 * s) % VOCAB for p in prompts], prefix))
    assert bd.status() == 0
    return got


@pytest.mark.parametrize("common", [256, 300, 17])
def test_forked_steps_match_separate_sequences(weights_2l, common):
    from paged import PrefixPlan
    prefix = _tokens(common, 1)
    prompts = [prefix + _tokens(1, 10 + i) for i in range(5)]
    plain = _decoder(weights_2l)
    plain.prefill_parallel(prompts)
    ref = _run(plain, prompts, 3)
    bd = _decoder(weights_2l)
    bd.prefill_parallel([prefix + [0]], seqs=[0])
    bd.fork(0, [1, 2, 3, 4], common)
    assert bd.pages_in_use == -(-common // 128) + 4 * (common % 128 > 0)
    plan = PrefixPlan([5], [common], 16, 8, 128, max_length=common + 8)
    _close(weights_2l, _run(bd, prompts, 3, plan), ref)
    assert plan.status() == 0
    # The split attention over the same shared pages: the same bits as without sharing.
    again = _decoder(weights_2l)
    again.prefill_parallel([prefix + [0]], seqs=[0])
    again.fork(0, [1, 2, 3, 4], common)
    for (t, n), (u, m) in zip(_run(again, prompts, 3), ref):
        assert t == u and torch.equal(n, m)


def test_groups_of_different_prefixes(weights_2l):
    from paged import PrefixPlan
    a, b = _tokens(200, 2), _tokens(129, 3)
    prompts = [a + _tokens(1, 20), a + _tokens(1, 21), b + _tokens(1, 22), b + _tokens(1, 23), b + _tokens(1, 24),
               _tokens(40, 25)]
    plain = _decoder(weights_2l)
    plain.prefill_parallel(prompts)
    ref = _run(plain, prompts, 2)
    bd = _decoder(weights_2l)
    bd.prefill_parallel([a + [0], b + [0], prompts[5]], seqs=[0, 2, 5])
    bd.fork(0, [1], 200)
    bd.fork(2, [3, 4], 129)
    plan = PrefixPlan([2, 3, 1], [200, 129, 0], 16, 8, 128, max_length=260)
    _close(weights_2l, _run(bd, prompts, 2, plan), ref)


def test_copy_on_write_keeps_the_siblings(weights_2l):
    """A child that goes back into shared pages writes into copies."""
    prefix = _tokens(256, 4)
    bd = _decoder(weights_2l)
    bd.prefill_parallel([prefix + [0]], seqs=[0])
    bd.fork(0, [1], 256)
    before = bd.k_pool[bd.page_table[0, :2].long()].clone()
    other = _tokens(30, 5)
    bd.reserve(1, 129, write_from=100)
    bd.prefill_parallel([other + [0]], seqs=[1], starts=[100])
    assert torch.equal(bd.k_pool[bd.page_table[0, :2].long()], before)
    plain = _decoder(weights_2l)
    plain.prefill_parallel([prefix[:100] + other + [0]], seqs=[1])
    x, y = _step(bd, [1], [130], [9]), _step(plain, [1], [130], [9])
    assert x[0] == y[0] and torch.equal(x[1], y[1])


def test_compaction_moves_what_is_in_use(weights_2l):
    prompts = [_tokens(n, 30 + n) for n in (300, 140, 260, 20)]
    bd = _decoder(weights_2l)
    bd.prefill_parallel(prompts)
    plain = _decoder(weights_2l)
    plain.prefill_parallel(prompts)
    bd.fork(2, [4], 259)
    bd.release([0, 3])
    assert bd.compact() > 0
    used = bd.pages_in_use
    assert int(bd.page_table.max()) < used and bd.page_table.cpu().tolist() == bd.pages.table
    for s in (1, 2):
        x = _step(bd, [s], [len(prompts[s]) - 1], [prompts[s][-1]])
        y = _step(plain, [s], [len(prompts[s]) - 1], [prompts[s][-1]])
        assert x[0] == y[0] and torch.equal(x[1], y[1])
    bd.reserve(0, 0)
    assert bd.pages.table[0][0] == used                # the first free page


def test_release_refuses_before_it_changes_anything(weights_2l):
    bd = _decoder(weights_2l)
    bd.reserve(1, 200)
    for bad in ([1, 6], [1, -7], 6):
        with pytest.raises(IndexError):
            bd.release(bad)
        assert bd.pages_in_use == 2 and bd.page_table.cpu().tolist() == bd.pages.table
    bd.release(torch.tensor([1, 1]))
    assert bd.pages_in_use == 0 and int(bd.page_table.max()) == -1
    bd.reserve(5, 0)
    bd.release(-1)                                     # as an index of a list
    assert bd.pages_in_use == 0 and int(bd.page_table.max()) == -1


@pytest.mark.parametrize("sampled", [False, True])
def test_generate_shared(weights_2l, sampled):
    """Completions of one prompt and of prompts that begin alike: the greedy
    tokens of separate sequences as far as the logits' margins decide them."""
    from sampling import SamplingParams
    prefix = _tokens(200, 6)
    suffixes = [_tokens(n, 40 + n) for n in (3, 70, 1)]
    bd = _decoder(weights_2l)
    sp = SamplingParams(0.9, 20, 0.95, 3) if sampled else None
    got = bd.generate_shared(prefix, suffixes, 6, sampling=sp)
    assert bd.status() == 0 and [len(g) for g in got] == [6] * 3
    bd.release([0, 1, 2])
    assert bd.pages_in_use == 0
    assert bd.generate_shared(prefix, suffixes, 6, sampling=sp) == got
    bd.release([0, 1, 2])
    same = bd.generate_shared(prefix, [[], [], [], []], 5, sampling=sp)
    if sampled:
        assert len({tuple(t) for t in same}) > 1        # random streams of their own
        return
    assert same == [same[0]] * 4
    # Replay along the generated tokens without sharing.
    emb = weights_2l["embed_weight"].cuda()
    plain = _decoder(weights_2l)
    full = [prefix + s + g[:-1] for s, g in zip(suffixes, got)]
    plain.prefill_parallel([f + [0] for f in full])
    for i, (s, g) in enumerate(zip(suffixes, got)):
        for k in range(len(g)):
            pos = len(prefix) + len(s) - 1 + k
            _, norm = _step(plain, [i], [pos], [full[i][pos]])
            logits = logits_from_norm(norm[0], emb)
            assert float(logits.max() - logits[g[k]]) <= 2 * LOGIT_ATOL


def test_captured_step(weights_2l):
    from paged import PrefixPlan
    prefix = _tokens(300, 7)
    bd = _decoder(weights_2l)
    bd.prefill_parallel([prefix + [0]], seqs=[0])
    bd.fork(0, [1, 2], 300)
    for i in range(3):
        bd.reserve(i, 300)
    plan = PrefixPlan([3], [300], 16, 8, 128, max_length=310)
    dev = dict(dtype=torch.int32, device=bd.dev)
    ids, pos, tok = torch.arange(3, **dev), torch.full((3,), 300, **dev), torch.tensor([5, 6, 7], **dev)
    norm = torch.empty(3, 1024, dtype=torch.float32, device=bd.dev)
    out = torch.empty(3, **dev)
    bd.step(ids, pos, tok, 300, norm_out=norm, out=out, prefix=plan)
    want = (out.clone(), norm.clone())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        bd.step(ids, pos, tok, 300, norm_out=norm, out=out, prefix=plan)
    norm.zero_()
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(norm, want[1])


def test_refusals(weights_2l):
    from batched import BatchedDecoder
    from paged import PrefixPlan
    flat = BatchedDecoder(weights_2l, num_seqs=2, num_layers=2)
    z = torch.zeros(2, dtype=torch.int32, device=flat.dev)
    plan = PrefixPlan([2], [16], 16, 8, 128, max_length=64)
    with pytest.raises(ValueError, match="paged"):
        flat.step(z, z, z, 0, prefix=plan)
    with pytest.raises(ValueError, match="paged"):
        flat.fork(0, [1], 1)
    with pytest.raises(ValueError, match="paged"):
        flat.compact()
    bd = _decoder(weights_2l)
    with pytest.raises(ValueError, match="the step has 2 rows"):
        bd.step(z, z, z, 0, prefix=PrefixPlan([3], [16], 16, 8, 128, max_length=64))
    with pytest.raises(ValueError, match="heads"):
        bd.step(z, z, z, 0, prefix=PrefixPlan([2], [16], 8, 8, 128, max_length=64))
    with pytest.raises(RuntimeError, match="max_length"):
        bd.step(z, z, z, 0, prefix=PrefixPlan([2], [16], 16, 8, 128, max_length=4000))
    with pytest.raises(ValueError, match="no page"):
        bd.fork(0, [1], 5)
    with pytest.raises(ValueError, match="past max_seq"):
        bd.generate_shared([1, 2], [[], []], 5000)
    with pytest.raises(ValueError, match="none of them empty"):
        bd.generate_shared([], [[], []], 5)
    bd.reserve(1, 3)
    with pytest.raises(ValueError, match="hold no pages"):
        bd.generate_shared([1, 2], [[], []], 5)
