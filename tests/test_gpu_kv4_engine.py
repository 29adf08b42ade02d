"""The engine with a 4-bit key/value cache, and forks of sequences: a small Qwen3 against its own layers over unquantised keys and values, and every
way of running the same tokens against the others."""
import pytest
import torch

import nanoquantization_b200 as nq
from nanoquantization_b200.engine import LLMEngine, Sequence
from nanoquantization_b200.models import Qwen3QuantizedForCausalLM

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _model(dtype=torch.bfloat16, seed=0, heads=8, kv_heads=2):
    torch.manual_seed(seed)
    m = Qwen3QuantizedForCausalLM(2, 512, 256, heads, kv_heads, 4096, 512, 4, 128, 128, False, 1e6, 1e-6, device=DEV, dtype=dtype)
    g = torch.Generator(device=DEV).manual_seed(seed)
    for mod in m.modules():
        if isinstance(mod, nq.WQLinear_GEMM):
            mod.qweight.copy_(torch.randint(-2 ** 31, 2 ** 31, mod.qweight.shape, generator=g, device=DEV, dtype=torch.int64).to(torch.int32))
            mod.qzeros.copy_(torch.randint(-2 ** 31, 2 ** 31, mod.qzeros.shape, generator=g, device=DEV, dtype=torch.int64).to(torch.int32))
            mod.qscales.copy_((torch.rand(mod.qscales.shape, generator=g, device=DEV) * 9e-3 + 1e-3).to(dtype))
    m.fuse_projections()
    return m


def _tokens(n, seed):
    return torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _engine(m, **kw):
    return LLMEngine(m, **{"num_blocks": 64, "block_size": 16, "max_batch": 8, "kv_bits": 4, **kw})


def _rel(a, b):
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@torch.no_grad()
def test_generation_graphs_match_eager_and_blocks_come_back(dtype):
    m = _model(dtype, 1)
    prompts = [_tokens(n, n) for n in (5, 133, 17, 1)]
    runs = []
    for kw in ({"use_cuda_graph": False}, {}, {"block_size": 48, "num_blocks": 30}, {"num_blocks": 16, "max_batch": 3}):      # the last one has to preempt
        e = _engine(m, **kw)
        runs.append(e.generate(prompts, 40))
        assert len(e.blocks.free) == kw.get("num_blocks", 64) and not e.blocks.shared
    assert all(len(o) == 40 for o in runs[0])
    # greedy tokens of a random model: the first ones have to agree, later ones may part where two logits are within rounding
    for r in runs[1:]:
        assert [o[0] for o in r] == [o[0] for o in runs[0]]
    assert runs[0] == runs[1]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@torch.no_grad()
def test_logits_do_not_depend_on_how_the_tokens_came(dtype):
    """Whole, in portions, token by token: the cache holds the same rows but where a rounding decides a level."""
    m = _model(dtype, 2)
    tokens = _tokens(150, 9)
    want = _engine(m).extend([(Sequence(0, [], 1 << 30), tokens, range(150))])[0]
    e, s, got = _engine(m), Sequence(0, [], 1 << 30), []
    for a, b in ((0, 70), (70, 71), (71, 76), (76, 140)):
        got.append(e.extend([(s, tokens[a:b], range(b - a))])[0])
    for i in range(140, 150):
        got.append(e.extend([(s, tokens[i:i + 1], [0])])[0])
    got = torch.cat(got)
    assert torch.isfinite(want).all() and _rel(got, want) <= (0.02 if dtype == torch.float16 else 0.06)
    # and they are near those of an unquantised cache: a level is off by a thirtieth of a group's range at most
    full = _engine(m, kv_bits=16).extend([(Sequence(0, [], 1 << 30), tokens, range(150))])[0]
    assert _rel(want, full) <= 0.35


@torch.no_grad()
def test_prompts_in_portions_beside_whole_ones():
    m = _model(torch.float16, 6)
    prompts = [_tokens(n, 70 + n) for n in (300, 9, 120, 64)]
    whole = _engine(m, num_blocks=80).generate(prompts, 3)
    for portion in (50, 128, 1):
        e = _engine(m, num_blocks=80, prefill_portion=portion)
        got = e.generate(prompts if portion > 1 else prompts[1:2], 3)
        assert [o[0] for o in got] == [o[0] for o in (whole if portion > 1 else whole[1:2])] and len(e.blocks.free) == 80


@torch.no_grad()
def test_forks_of_a_full_cache_are_refused_and_leave_it_as_it_was():
    m = _model(torch.float16, 7)
    e = _engine(m, num_blocks=4)
    s = Sequence(0, [], 1 << 30)
    e.extend([(s, _tokens(60, 3), [])])                # four blocks, the last one not full
    t = e.fork(s)
    with pytest.raises(RuntimeError, match="cannot hold"):
        e.extend([(t, [5], [0])])                      # no block is left for a copy
    assert t.blocks == s.blocks and not e.blocks.copies
    e.drop(t)
    assert torch.isfinite(e.extend([(s, [5], [0])])[0]).all() and not e.blocks.shared
    e.drop(s)
    assert sorted(e.blocks.free) == [0, 1, 2, 3]


@pytest.mark.parametrize("bits", [16, 4])
@torch.no_grad()
def test_forks_go_on_as_their_sequences_would(bits):
    m = _model(seed=3)
    prefix, tails = _tokens(37, 4), [_tokens(n, 50 + n) for n in (1, 5, 30, 3)]
    e = _engine(m, kv_bits=bits)
    s = Sequence(0, [], 1 << 30)
    e.extend([(s, prefix, [])])
    forks = [e.fork(s) for _ in tails[1:]]
    used = 64 - len(e.blocks.free)
    assert used == 3                                   # nothing copied yet
    mine = [s] + forks
    got = e.extend([(q, t, range(len(t))) for q, t in zip(mine, tails)])
    more = e.extend([(q, [7], [0]) for q in mine])     # one token each: the decode path
    for t, a, b in zip(tails, got, more):
        f = _engine(m, kv_bits=bits)
        alone = Sequence(0, [], 1 << 30)
        f.extend([(alone, prefix, [])])
        want = f.extend([(alone, t, range(len(t)))])[0]
        assert _rel(a, want) <= 0.03 and _rel(b, f.extend([(alone, [7], [0])])[0]) <= 0.03
    assert len({q.blocks[2] for q in mine}) == 4 and len({q.blocks[0] for q in mine}) == 1
    grandchild = e.fork(forks[1])
    e.drop(forks[1])
    a, b = e.extend([(grandchild, [9], [0]), (s, [9], [0])])
    assert torch.isfinite(a).all() and torch.isfinite(b).all()
    for q in [s, grandchild] + forks[:1] + forks[2:]:
        e.drop(q)
    assert sorted(e.blocks.free) == list(range(64)) and not e.blocks.shared
    e._check_device_status()


@torch.no_grad()
def test_forks_of_recurrent_models_copy_their_states():
    import vemedra_cases as C
    c = C.config()
    model = C.build(c, C.weights(c, 7), DEV, torch.float32)
    tokens = [3, 1, 4, 1, 5, 9, 2, 6]
    e = LLMEngine(model, num_blocks=40, block_size=8, max_batch=4)
    s = Sequence(0, [], 1 << 30)
    e.extend([(s, tokens, [])])
    t = e.fork(s)
    assert t.slot != s.slot
    a = e.extend([(s, [5, 3], [0, 1])])[0]
    b = e.extend([(t, [5, 3], [0, 1])])[0]             # the first one's step has not touched it
    assert torch.equal(a, b)
    others = [e.fork(t) for _ in range(2)]
    with pytest.raises(RuntimeError, match="no state slot"):
        e.fork(t)
    for q in [s, t] + others:
        e.drop(q)
    assert sorted(e.blocks.free) == list(range(40))


def test_commands_take_the_cache_and_forks(tmp_path):
    """Generation with a 4-bit cache, and a replay in which one request goes on from another."""
    import json
    import os
    import subprocess
    import sys
    import numpy as np
    from safetensors.torch import save_file
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    torch.manual_seed(5)
    m = Qwen3QuantizedForCausalLM(1, 256, 256, 4, 2, 512, 256, 4, 128, 128, False, 1e6, 1e-6, device="cpu", dtype=torch.float16)
    for mod in m.modules():
        if isinstance(mod, nq.WQLinear_GEMM):
            mod.qweight.copy_(torch.randint(-2 ** 31, 2 ** 31, mod.qweight.shape, dtype=torch.int64).to(torch.int32))
            mod.qzeros.copy_(torch.randint(-2 ** 31, 2 ** 31, mod.qzeros.shape, dtype=torch.int64).to(torch.int32))
            mod.qscales.copy_((torch.rand(mod.qscales.shape) * 9e-3 + 1e-3).half())
    (tmp_path / "m").mkdir()
    save_file({k: v.contiguous() for k, v in m.state_dict().items()}, str(tmp_path / "m" / "model.safetensors"))
    config = {"architectures": ["Qwen3ForCausalLM"], "num_hidden_layers": 1, "vocab_size": 256, "hidden_size": 256, "num_attention_heads": 4, "num_key_value_heads": 2,
              "max_position_embeddings": 512, "intermediate_size": 256, "head_dim": 128, "rope_theta": 1e6, "rms_norm_eps": 1e-6,
              "quantization_config": {"w_bits": 4, "group_size": 128}}
    (tmp_path / "m" / "config.json").write_text(json.dumps(config))
    cmd = [sys.executable, "-m", "nanoquantization_b200.cli"]
    gen = subprocess.run(cmd + ["generate", "--model", str(tmp_path / "m"), "--dtype", "float16", "--kv-bits", "4", "--max-new-tokens", "5"],
                         input="5 17 3\n8 8\n", capture_output=True, text=True, cwd=root)
    assert gen.returncode == 0, gen.stderr
    assert [len(line.split()) for line in gen.stdout.splitlines()] == [5, 5]
    steps = [{"step": 0, "entries": [{"id": "a", "tokens": [5, 17, 3, 9], "want": []}]},
             {"step": 1, "entries": [{"id": "a", "tokens": [1, 2], "want": [0, 1]}, {"id": "b", "from": "a", "tokens": [1, 2], "want": [0, 1]}]},
             {"step": 2, "entries": [{"id": "b", "tokens": [4], "want": [0]}, {"id": "a", "tokens": [4], "want": [0]}], "end": ["a", "b"]}]
    out = tmp_path / "out"
    out.mkdir()
    run = subprocess.run(cmd + ["trace", "--model", str(tmp_path / "m"), "--dtype", "float16", "--kv-bits", "4", "--out", str(out)],
                         input="".join(json.dumps(s) + "\n" for s in steps), capture_output=True, text=True, cwd=root)
    assert run.returncode == 0, run.stderr
    assert run.stdout.split("\n")[:3] == ["done 0", "done 1", "done 2"]
    for i, n in ((1, 4), (2, 2)):
        logits = np.fromfile(out / f"{i}.f32", "<f4").reshape(n, 256)
        assert np.isfinite(logits).all() and np.array_equal(logits[:n // 2], logits[n // 2:])
