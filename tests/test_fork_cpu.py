"""Forks go on from where their sequences stand: what a step feeds the model, without a GPU (a forward that notes its inputs)."""
import pytest
import torch

from nanoquantization_b200.engine import LLMEngine, Sequence
from nanoquantization_b200.models.qwen3_quantized import Qwen3QuantizedForCausalLM


def _engine(**kw):
    model = Qwen3QuantizedForCausalLM(1, 64, 256, 2, 1, 32, 128, 4, 128, 128, device="cpu", dtype=torch.float16)
    engine = LLMEngine(model, **{"num_blocks": 12, "block_size": 4, "max_batch": 4, "use_cuda_graph": False, **kw})
    fed = []

    def forward(batch, decode, rows=None):
        fed.append((decode, batch.tokens.tolist(), batch.positions.tolist(), batch.cu.tolist(), None if rows is None else rows.tolist()))
        # a hidden state that names its position and token
        h = torch.stack([batch.positions.float(), batch.tokens.float()], -1)
        return h if rows is None else h[rows]
    engine._forward = forward
    model.logits = lambda h: h.clone()
    model.greedy_tokens = lambda h: torch.full((len(h),), 42)
    engine._check_device_status = lambda: None
    return engine, fed


def test_a_fork_of_a_sequence_that_is_generating():
    engine, fed = _engine()
    engine.add_request([1, 2, 3, 4, 5, 6], 10)
    engine.step(), engine.step()
    s = engine.scheduler.running[0]
    assert s.output == [42, 42] and s.computed == 7
    t, u = engine.fork(s), engine.fork(s)
    fed.clear()
    out = engine.extend([(t, [33], [0])])[0]
    # its newest token has not been through the model: it comes first, at position 7
    assert fed == [(False, [42, 33], [7, 8], [0, 2], [1])] and out.tolist() == [[8.0, 33.0]]
    assert (t.prompt, t.output, t.computed) == ([1, 2, 3, 4, 5, 6, 42, 42, 33], [], 9)
    fed.clear()
    out = engine.extend([(t, [34], [0]), (u, [7, 8], [1])])
    assert fed == [(False, [34, 42, 7, 8], [9, 7, 8, 9], [0, 1, 4], [0, 3])]
    assert out[0].tolist() == [[9.0, 34.0]] and out[1].tolist() == [[9.0, 8.0]]
    fed.clear()
    out = engine.extend([(t, [35], [0]), (u, [9], [0])])      # nothing is left over: the decode path
    assert fed == [(True, [35, 9], [10, 10], [0, 1, 2], None)]
    # the first one goes on as if nothing had been
    fed.clear()
    engine.step()
    assert fed == [(True, [42], [7], [0, 1], None)] and s.output == [42] * 3 and s.prompt == [1, 2, 3, 4, 5, 6]
    while engine.scheduler.running:
        done = engine.step()
    assert done[0].carried + done[0].output == [42] * 10
    # what a fork has generated stays with it
    assert t.carried == [42, 42] and t.max_new_tokens == 8
    engine.drop(t), engine.drop(u)
    assert sorted(engine.blocks.free) == list(range(12)) and not engine.blocks.shared


def test_a_fork_of_a_sequence_that_waits():
    """In the middle of its prompt, and with nothing computed."""
    engine, fed = _engine(prefill_portion=4)
    engine.add_request([1, 2, 3, 4, 5, 6], 10)
    waiting = engine.fork(engine.scheduler.waiting[0])
    engine.step()
    s = engine.scheduler.waiting[0]
    assert s.computed == 4
    t = engine.fork(s)
    fed.clear()
    out = engine.extend([(t, [33, 34], [0, 1]), (waiting, [9], [0])])
    assert fed[0][1:4] == ([5, 6, 33, 34, 1, 2, 3, 4, 5, 6, 9], [4, 5, 6, 7, 0, 1, 2, 3, 4, 5, 6], [0, 4, 11])
    assert out[0].tolist() == [[6.0, 33.0], [7.0, 34.0]] and out[1].tolist() == [[6.0, 9.0]]


def test_no_tokens_are_given_but_one_is_left():
    engine, fed = _engine()
    engine.add_request([1, 2, 3], 10)
    engine.step()
    t = engine.fork(engine.scheduler.running[0])
    fed.clear()
    assert engine.extend([(t, [], [])]) == [None]
    assert fed == [(True, [42], [3], [0, 1], None)] and t.computed == len(t) == 4


def test_steps_that_are_refused():
    engine, fed = _engine()
    engine.add_request([1, 2, 3], 10)
    with pytest.raises(ValueError, match="the scheduler runs"):
        engine.extend([(engine.scheduler.waiting[0], [5], [0])])
    engine.step()
    s = engine.scheduler.running[0]
    fed.clear()
    with pytest.raises(ValueError, match="the scheduler runs"):
        engine.extend([(s, [5], [0])])
    t = engine.fork(s)
    with pytest.raises(ValueError, match="twice"):
        engine.extend([(t, [5], [0]), (t, [6], [0])])
    assert not fed and t.prompt == [1, 2, 3] and t.output == [42]


def test_a_step_that_the_cache_cannot_hold_leaves_the_tokens_out():
    engine, fed = _engine(num_blocks=2)
    s = Sequence(0, [], 1 << 30)
    engine.extend([(s, [1, 2, 3, 4, 5], [])])
    with pytest.raises(RuntimeError, match="cannot hold"):
        engine.extend([(s, [6, 7, 8, 9], [])])
    assert s.prompt == [1, 2, 3, 4, 5]
    fed.clear()
    engine.extend([(s, [6], [0])])
    assert fed == [(True, [6], [5], [0, 1], None)]
