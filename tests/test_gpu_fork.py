"""Forks of sequences that the engine is generating, against fresh sequences with the same tokens."""
import pytest
import torch

from nanoquantization_b200.engine import Sequence
from test_gpu_kv4_engine import _engine, _model, _rel, _tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("graph", [False, True])
@torch.no_grad()
def test_forks_in_the_middle_of_generation(graph, bits):
    m = _model(torch.float16, 8)
    prompts = [_tokens(n, 90 + n) for n in (37, 5, 100)]
    want = _engine(m, kv_bits=bits, use_cuda_graph=graph).generate(prompts, 20)
    e = _engine(m, kv_bits=bits, use_cuda_graph=graph, max_batch=16)      # nine at a time
    for p in prompts:
        e.add_request(p, 20)
    for _ in range(8):
        e.step()
    running = list(e.scheduler.running)
    assert [s.output for s in running] == [w[:8] for w in want]
    tails = [[7], [3, 1, 4], [9, 9]]
    forks = [e.fork(s) for s in running]
    got = [e.extend([(t, x, range(len(x)))])[0] for t, x in zip(forks, tails)]
    together = [e.fork(s) for s in running]
    both = e.extend([(t, x, range(len(x))) for t, x in zip(together, tails)])
    more = e.extend([(t, [11], [0]) for t in together])          # the decode path
    for p, w, x, a, b, c in zip(prompts, want, tails, got, both, more):
        f, alone = _engine(m, kv_bits=bits, use_cuda_graph=graph), Sequence(0, [], 1 << 30)
        f.extend([(alone, p, [])])
        for y in w[:7]:                                          # as they came: one at a time
            f.extend([(alone, [y], [])])
        ref = f.extend([(alone, w[7:8] + x, range(1, 1 + len(x)))])[0]
        assert _rel(a, ref) <= 0.02 and _rel(b, ref) <= 0.02
        assert _rel(c, f.extend([(alone, [11], [0])])[0]) <= 0.02
    # and those that were forked go on as they would have
    done = []
    while e.scheduler.running:
        done += e.step()
    assert [s.carried + s.output for s in sorted(done, key=lambda s: s.seq_id)] == want
    for t in forks + together:
        e.drop(t)
    assert sorted(e.blocks.free) == list(range(64)) and not e.blocks.shared
