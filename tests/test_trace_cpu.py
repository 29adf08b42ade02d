"""The replay of given tokens and the steps that it runs on, without a GPU: what reaches the disk, and what is refused."""
import io
import json

import pytest
import torch

import nanoquantization_b200.engine as engine_module
from nanoquantization_b200 import _lib, cli


class _Engine:
    """Takes the engine's place: logits that name the step's tokens, and a status that fails when it is told to."""
    fails = False

    def __init__(self, model, **kw):
        self.live = []

    def extend(self, entries):
        for s, tokens, _ in entries:
            s.prompt.extend(tokens)
        return [torch.tensor([[float(t[w]), float(len(s))] for w in want]) if want else None for s, t, want in entries]

    def fork(self, s):
        return engine_module.Sequence(s.seq_id, list(s.prompt), s.max_new_tokens)

    def drop(self, s):
        pass

    def _check_device_status(self):
        if self.fails:
            raise RuntimeError("a bounded device-side wait timed out")


@pytest.fixture
def trace(monkeypatch, tmp_path):
    monkeypatch.setattr(engine_module, "LLMEngine", _Engine)
    monkeypatch.setattr(cli, "_model", lambda args: (object(), None))
    monkeypatch.setattr("nanoquantization_b200.csrc.build.build_library", lambda path: path)

    def run(*steps):
        monkeypatch.setattr("sys.stdin", io.StringIO("".join(json.dumps({"step": i, **s}) + "\n" for i, s in enumerate(steps))))
        return cli.main(["trace", "--model", "none", "--out", str(tmp_path)])
    run.out = tmp_path
    return run


def test_logits_of_a_step_that_gave_up_are_not_written(trace, monkeypatch, capsys):
    steps = [{"entries": [{"id": "a", "tokens": [5, 6], "want": [1]}]}, {"entries": [{"id": "a", "tokens": [7], "want": [0]}]}]
    assert trace(*steps) == 0 and sorted(p.name for p in trace.out.iterdir()) == ["0.f32", "1.f32"]
    for p in list(trace.out.iterdir()):
        p.unlink()
    monkeypatch.setattr(_Engine, "fails", True)
    capsys.readouterr()
    with pytest.raises(RuntimeError, match="timed out"):
        trace(*steps)
    assert not list(trace.out.iterdir()) and "done" not in capsys.readouterr().out


@pytest.mark.parametrize("n", [1, 3])
def test_a_bad_index_ends_the_step_that_met_it(n, monkeypatch):
    """Both ways that given tokens take."""
    from nanoquantization_b200.engine import LLMEngine, Sequence
    from nanoquantization_b200.models.qwen3_quantized import Qwen3QuantizedForCausalLM
    model = Qwen3QuantizedForCausalLM(1, 64, 256, 2, 1, 32, 128, 4, 128, 128, device="cpu", dtype=torch.float16)
    engine = LLMEngine(model, num_blocks=4, block_size=16, max_batch=2, use_cuda_graph=False, kv_bits=4)
    word = torch.zeros(1, dtype=torch.int32)

    def forward(batch, decode, rows=None):
        if batch.tokens[0] == 9:
            word[0] = 10
        return torch.zeros(len(batch.tokens) if rows is None else len(rows), 2)
    engine._forward = forward
    model.logits = lambda h: h
    model.greedy_tokens = lambda h: None
    monkeypatch.setattr(_lib, "_cache_status", {0: word})
    s = Sequence(0, [], 1 << 30)
    engine.extend([(s, [1, 2, 3], [])])
    with pytest.raises(RuntimeError, match="outside its buffer"):
        engine.extend([(s, [9] * n, [0])])
    assert not word.any()
    engine.extend([(s, [1] * n, [0])])


def test_requests_that_go_on_from_others(trace, capsys):
    start = {"entries": [{"id": "a", "tokens": [5, 6]}]}
    assert trace(start, {"entries": [{"id": "b", "from": "a", "tokens": [7], "want": [0]}, {"id": "a", "tokens": [8]}], "end": ["a"]},
                 {"entries": [{"id": "c", "from": "b", "tokens": [9]}]}) == 0
    assert capsys.readouterr().out.split() == ["done", "0", "done", "1", "done", "2"]
    # a request that is not there, that ended, that starts in the same step; one that lives already, or that the step has forked
    for step in ({"entries": [{"id": "b", "from": "x", "tokens": [7]}]}, {"entries": [{"id": "a", "from": "a", "tokens": [7]}]},
                 {"entries": [{"id": "b", "tokens": [7]}, {"id": "c", "from": "b", "tokens": [7]}]},
                 {"entries": [{"id": "b", "from": "a", "tokens": [7]}, {"id": "c", "from": "b", "tokens": [7]}]},
                 {"entries": [{"id": "b", "from": "a", "tokens": [7]}, {"id": "b", "from": "a", "tokens": [7]}]}):
        assert trace(start, step) == 2
        got = capsys.readouterr()
        assert got.out.split() == ["done", "0"] and '"from"' in got.err and "step 1" in got.err
    assert trace({**start, "end": ["a"]}, {"entries": [{"id": "b", "from": "a", "tokens": [7]}]}) == 2
