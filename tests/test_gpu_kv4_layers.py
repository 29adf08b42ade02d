"""The engine with a 4-bit cache against its own layers over keys and values that are quantised as described, in 64 bits, and kept by sequence: not
through the engine's blocks, tables and rows.

The two differ by roundings of half a step u a layer; where one moves a key or a value of the next layer over the middle between two levels (0.4 of a
standard deviation apart), it changes by all of that: for 2 u that is sqrt(5 u) * 0.4, 0.02 for float16 and 0.06 for bfloat16, of a layer's keys and
values, and no more than that of the logits."""
import pytest
import torch

from nanoquantization_b200.engine import Sequence
from nanoquantization_b200.models.qwen3_quantized import Qwen3QuantizedAttention
from test_gpu_kv4_engine import _engine, _model, _rel, _tokens
from tests import kv4_reference as ref

pytestmark = pytest.mark.gpu


class _Plain:
    """Takes the kernels' place: ``who`` names the sequences of the step, ``kept`` holds their keys and values by layer."""

    def __init__(self):
        self.who, self.kept = [], {}

    def attend(self, attn, qkv, positions, k_cache, v_cache, batch, decode):
        dtype, hq, hk, o, out = qkv.dtype, attn.num_heads, attn.num_kv_heads, 0, []
        for name, n in zip(self.who, batch.lens):
            x = qkv[o:o + n].double().view(n, hq + 2 * hk, 128)
            k, v = self.kept.get((id(attn), name), (x[:0, :hk], x[:0, :hk]))
            at = torch.arange(len(k), len(k) + n, device=qkv.device)
            turn = lambda y, w: ref.norm_rope(y, w, attn.rope.cos_sin_cache, at, attn.q_norm.eps)  # noqa: E731
            k = torch.cat([k, ref.quantised(turn(x[:, hq:hq + hk], attn.k_norm.weight), dtype)])
            v = torch.cat([v, ref.quantised(x[:, hq + hk:], dtype)])
            self.kept[id(attn), name] = k, v
            out.append(ref.attend(turn(x[:, :hq], attn.q_norm.weight), k, v, len(k) - n).flatten(1))
            o += n
        return torch.cat(out).to(dtype)

    def fork(self, old, new):
        self.kept.update({(a, new): kv for (a, name), kv in self.kept.items() if name == old})


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@torch.no_grad()
def test_the_engine_against_layers_over_quantised_keys_and_values(dtype, graph, monkeypatch):
    m, plain = _model(dtype, 11), _Plain()
    steps = [{"a": 150, "b": 9}, {"a": 1, "b": 1}, {"b": 40, "c": 1, "a": 3}, {"a": 1, "b": 1, "c": 1, "d": 1}, {"d": 20, "c": 1}, {"d": 1}]
    forks = {2: ("a", "c"), 3: ("b", "d")}          # ahead of a step
    runs = []
    for kernels in (True, False):
        e, live, logits = _engine(m, use_cuda_graph=graph and kernels), {}, []
        with monkeypatch.context() as patch:
            if not kernels:
                patch.setattr(Qwen3QuantizedAttention, "_attend_kv4", lambda self, *args: plain.attend(self, *args))
            for i, step in enumerate(steps):
                if i in forks:
                    old, new = forks[i]
                    live[new] = e.fork(live[old])
                    plain.fork(old, new)
                plain.who = list(step)
                logits.append(e.extend([(live.setdefault(w, Sequence(0, [], 1 << 30)), _tokens(n, 7 * i + ord(w)), range(n)) for w, n in step.items()]))
        runs.append(logits)
    for mine, want in zip(*runs):
        for a, b in zip(mine, want):
            assert torch.isfinite(a).all() and _rel(a, b) <= (0.02 if dtype == torch.float16 else 0.06)
