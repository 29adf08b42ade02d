"""The 4-bit cache and copies of pages without a GPU: refusals at the C entries and in Python, and the layout's own reference."""
import ctypes

import pytest
import torch

from nanoquantization_b200 import _lib
from nanoquantization_b200.layers import kv4, pages
from tests import kv4_reference as ref


def _c(pages_=4, heads=2, block=16, k=1 << 20, v=1 << 20):
    return _lib.Kv4(k, v, pages_, heads, block)


P = 1 << 20        # an address that is aligned and never reached


def test_refusals_of_the_store_and_the_read_back():
    lib = _lib.load()

    def store(cache=None, qkv=P, stride=8 * 128, qw=P, cs=P, maxpos=10, rows=P, out=P, T=1, heads=4, dtype=0):
        return lib.nqb200_kv4_store(qkv, stride, qw, P, cs, maxpos, P, rows, cache or _c(), out, T, heads, 1e-6, dtype, None, None)
    assert lib.nqb200_kv4_store(P, 1024, P, P, P, 10, P, P, None, P, 1, 4, 1e-6, 0, None, None) == 4
    for bad in (_c(0), _c(-1), _c(1 << 31), _c(heads=0), _c(heads=4097), _c(block=0), _c(block=24), _c(block=-16)):
        assert store(bad) == 1
        assert lib.nqb200_kv4_load(bad, P, P, P, 1, 0, None, None) == 1
    assert store(_c(k=None)) == store(_c(v=0)) == 4 and store(_c(k=P + 8)) == 3
    assert store(T=-1) == store(heads=0) == store(maxpos=0) == store(stride=8 * 128 - 4) == store(stride=8 * 128 + 2) == 1
    assert store(dtype=2) == store(dtype=-1) == 2
    assert store(T=0, qkv=None) == 0 and store(T=1 << 31) == 9
    assert store(qkv=None) == store(qw=None) == store(cs=None) == store(rows=None) == store(out=None) == 4
    assert store(qkv=P + 4) == store(qw=P + 2) == store(cs=P + 8) == store(out=P + 4) == 3

    def load(n=1, rows=P, k=P, v=P, dtype=0):
        return lib.nqb200_kv4_load(_c(), rows, k, v, n, dtype, None, None)
    assert load(-1) == 1 and load(dtype=2) == 2 and load(0, None) == 0 and load(1 << 31) == 9
    assert load(rows=None) == load(k=None) == load(v=None) == 4 and load(k=P + 8) == load(v=P + 8) == 3


def test_refusals_of_the_attention():
    lib = _lib.load()

    def decode(cache=None, qkv=P, stride=8 * 128, maxpos=10, rows=P, table=P, width=3, ctx=P, out=P, batch=1, heads=4, dtype=0, scratch=P, nbytes=1 << 40):
        return lib.nqb200_kv4_decode_attention(qkv, stride, P, P, P, maxpos, P, rows, cache or _c(), table, width, ctx, out, batch, heads, 0.1, 1e-6, dtype, scratch, nbytes, None, None)
    assert decode(_c(block=8)) == decode(heads=3) == decode(heads=0) == decode(width=0) == decode(width=1 << 31) == decode(batch=-1) == decode(batch=65536) == 1
    assert decode(stride=7 * 128) == decode(stride=8 * 128 + 4) == decode(maxpos=0) == 1
    assert decode(dtype=2) == 2 and decode(batch=0, qkv=None) == 0
    assert decode(qkv=None) == decode(rows=None) == decode(table=None) == decode(ctx=None) == decode(out=None) == 4
    assert decode(qkv=P + 8) == decode(out=P + 8) == 3

    def prompt(cache=None, q=P, stride=512, table=P, width=3, cu=P, out=P, batch=1, T=4, max_len=4, max_ctx=4, tiles=1, heads=4, dtype=0, scratch=P, nbytes=1 << 40):
        return lib.nqb200_kv4_prompt_attention(q, stride, cache or _c(), table, width, cu, P, out, batch, T, max_len, max_ctx, tiles, heads, 0.1, dtype, scratch, nbytes, None, None)
    assert prompt(_c(block=8)) == prompt(heads=3) == prompt(width=0) == prompt(batch=-1) == prompt(batch=65536) == prompt(T=-1) == prompt(max_len=-1) == 1
    assert prompt(max_ctx=3) == prompt(tiles=-1) == prompt(stride=504) == prompt(stride=516) == 1
    assert prompt(dtype=7) == 2 and prompt(batch=0, q=None) == prompt(T=0, q=None) == 0
    assert prompt(q=None) == prompt(table=None) == prompt(cu=None) == prompt(out=None) == 4 and prompt(q=P + 8) == prompt(out=P + 8) == 3


def test_tables_whose_last_tile_would_pass_31_bits_are_refused():
    lib = _lib.load()
    for block in (16, 48, 256):
        most = (2**31 - 1 - 256) // block
        for width in (most + 1, (2**31 - 1) // block):
            assert lib.nqb200_kv4_decode_attention(P, 1024, P, P, P, 10, P, P, _c(block=block), P, width, P, P, 1, 4, 0.1, 1e-6, 0, P, 1 << 40, None, None) == 1
            assert lib.nqb200_kv4_prompt_attention(P, 512, _c(block=block), P, width, P, P, P, 1, 4, 4, 4, 1, 4, 0.1, 0, P, 1 << 40, None, None) == 1
            assert lib.nqb200_kv4_decode_scratch_bytes(width, block, 1, 4, 2) == 0
        assert lib.nqb200_kv4_decode_scratch_bytes(most, block, 1, 4, 2) > 0


def test_decode_steps_of_short_tables_need_no_scratch():
    need = _lib.load().nqb200_kv4_decode_scratch_bytes
    for block in (16, 48, 256):
        for batch in (1, 2, 3, 8, 100):
            for heads, kv_heads in ((1, 1), (8, 1), (32, 8), (64, 8)):
                width = kv4.SPLIT_KEYS // block
                assert need(width - (width * block >= kv4.SPLIT_KEYS), block, batch, heads, kv_heads) == 0
    assert need(16, 256, 1, 8, 1) > 0 and need(1 << 20, 16, 1, 8, 1) > 0
    for bad in ((0, 16, 1, 8, 1), (16, 0, 1, 8, 1), (16, 256, 0, 8, 1), (16, 256, 1, 9, 2), (16, 256, 1, 8, 0), (1 << 31, 16, 1, 8, 1)):
        assert need(*bad) == 0


def test_which_way_a_prompt_takes():
    name = _lib.load().nqb200_kv4_prompt_kernel_name
    assert name(1, 0, 1, 1, 1, 4, 2) == name(0, 1, 1, 1, 1, 4, 2) == name(1, 1, 1, 1, 1, 4, 3) == name(1, 2, 2, 1, 1, 4, 2) == b"invalid"
    for heads in (16, 32, 64):
        assert name(1, 16, 16, 16, 1, heads, 8) == name(4, 20, 5, 3006, 96, heads, 8) == b"rows"
        assert name(1, 8000, 8000, 8000, 63, heads, 8) == name(1, 500, 500, 12500, 98, heads, 8) == b"tiles_tcgen05"
    # 65536 columns of eight and more do not fit into the grid of the way for few rows
    assert name(1, 1 << 20, 1 << 20, 1 << 20, 1 << 13, 8, 8) == b"tiles_tcgen05"


def test_refusals_of_the_copies():
    lib = _lib.load()

    def copy(src, dst, rows=8, pools=(P,), nbytes=(16,)):
        n, m = len(src), len(pools)
        return lib.nqb200_copy_pages((ctypes.c_void_p * m)(*pools), (ctypes.c_int64 * m)(*nbytes), m, rows, (ctypes.c_int32 * n)(*src), (ctypes.c_int32 * n)(*dst), n, None)
    assert copy([], []) == 0 and copy([0], [1], pools=(), nbytes=()) == 0
    assert copy([0], [1], rows=0) == copy([0], [1], nbytes=(0,)) == 1 and copy([0], [1], pools=(None,)) == 4
    # out of range, a target twice, a target that is a source
    for src, dst in (([-1], [1]), ([8], [1]), ([0], [-1]), ([0], [8]), ([0, 2], [1, 1]), ([0, 1], [1, 2]), ([3], [3]), ([0] * 9, list(range(9)))):
        assert copy(src, dst) == 10
    assert lib.nqb200_copy_pages(None, None, 1, 8, None, None, 1, None) == 4


def test_refusals_in_python():
    with pytest.raises(ValueError, match="multiple of 16"):
        kv4.new_cache(2, 24, 1, "cpu")
    kc, vc = kv4.new_cache(2, 32, 3, "cpu")
    assert kc.shape == vc.shape == (2, 3, 32 * 72) and kc.dtype == torch.uint8 and not kc.any()
    x = torch.zeros(1, 9 * 128, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        kv4.load(kc, vc, torch.zeros(1, dtype=torch.int64), torch.float16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        kv4.prompt_attention(x, 9, kc, vc, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), [1], [0])
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        pages.copy_pages([kc], [0], [1])
    with pytest.raises(ValueError, match="1 sources and 2 targets"):
        pages.copy_pages([kc], [0], [1, 2])
    pages.copy_pages([], [], [])
    pages.copy_pages([kc], [], [])
    for bad in ((kc.float(), vc), (kc, vc[:, :2]), (kc[:, :, :-72], vc[:, :, :-72]), (kc.transpose(0, 1), vc.transpose(0, 1)), (kc[0], vc[0])):
        with pytest.raises((TypeError, ValueError), match="4-bit cache"):
            kv4._cache(*bad)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_the_layout_reads_back_what_it_packs(dtype):
    x = torch.randn(40, 128, generator=torch.Generator().manual_seed(0), dtype=torch.float64)
    assert torch.equal(ref.unpack(*ref.pack(x, dtype), dtype), ref.quantised(x, dtype))
    assert float((ref.quantised(x, dtype) - x).abs().max()) <= float(ref.params_of(x, dtype)[0].max()) * 0.6


def test_a_zero_filled_cache_reads_as_zeros():
    assert not ref.unpack(torch.zeros(3, 64, dtype=torch.uint8), torch.zeros(3, 8, dtype=torch.uint8), torch.float16).any()


# ------------------------------------------------------------------ blocks that sequences share
def _manager(blocks=8, size=4):
    from nanoquantization_b200.engine import BlockManager
    m, log = BlockManager(blocks, size), []
    m.copy = lambda pairs: log.append(list(pairs))
    return m, log


def test_a_shared_block_is_copied_before_one_writes_into_it():
    from nanoquantization_b200.engine import Sequence
    m, log = _manager()
    a, b = Sequence(0, [1] * 10, 9), Sequence(1, [1] * 10, 9)
    assert m.ensure(a, 10)
    a.computed = b.computed = 10
    m.share(a, b)
    assert b.blocks == a.blocks and len(m.free) == 5
    assert m.ensure(a, 11) and a.blocks[:2] == b.blocks[:2] and a.blocks[2] != b.blocks[2]      # the one with token 10 in it
    assert m.copies == [(b.blocks[2], a.blocks[2])] and not log
    assert m.ensure(b, 11) and len(m.copies) == 1                                               # the other has it to itself now
    m.flush()
    assert log == [[(b.blocks[2], a.blocks[2])]] and not m.copies
    m.release(a)
    assert len(m.free) == 5 and set(m.free).isdisjoint(b.blocks)
    m.release(b)
    assert sorted(m.free) == list(range(8)) and not m.shared


def test_blocks_that_hold_nothing_yet_are_replaced_and_not_copied():
    from nanoquantization_b200.engine import Sequence
    m, log = _manager()
    a, b = Sequence(0, [1] * 8, 9), Sequence(1, [1] * 8, 9)
    assert m.ensure(a, 9)                   # a block more than the eight tokens that there are
    a.computed = b.computed = 8
    m.share(a, b)
    assert m.ensure(b, 9) and b.blocks[2] != a.blocks[2] and not m.copies and len(m.free) == 4


def test_no_change_where_there_is_no_room_for_a_copy():
    from nanoquantization_b200.engine import Sequence
    m, log = _manager(3)
    a, b = Sequence(0, [1] * 10, 9), Sequence(1, [1] * 10, 9)
    assert m.ensure(a, 10)
    a.computed = b.computed = 10
    m.share(a, b)
    before = list(b.blocks)
    assert not m.ensure(b, 11) and b.blocks == before and not m.copies and m.shared == {x: 1 for x in before}
    m.release(a)
    assert not m.free and m.ensure(b, 11) and b.blocks == before


def test_copies_run_before_their_blocks_change_hands():
    from nanoquantization_b200.engine import Sequence
    m, log = _manager()
    seqs = [Sequence(i, [1] * 6, 9) for i in range(3)]
    assert m.ensure(seqs[0], 6)
    for s in seqs:
        s.computed = 6
    m.share(seqs[0], seqs[1]), m.share(seqs[0], seqs[2])
    assert all(m.ensure(s, 7) for s in seqs) and len(m.copies) == 2 and len({s.blocks[1] for s in seqs}) == 3
    pending = list(m.copies)
    m.release(seqs[1])                      # its blocks go back to the pool: the copies have run
    assert log == [pending] and not m.copies
    t = Sequence(4, [], 1)
    m.share(seqs[0], t)
    m.reclaim(seqs[0], 4)
    assert seqs[0].blocks[0] == -1 and t.blocks[0] >= 0 and t.blocks[0] not in m.free
    for s in (seqs[0], seqs[2], t):
        m.release(s)
    assert sorted(m.free) == list(range(8)) and not m.shared


def test_engines_that_a_4_bit_cache_is_not_for():
    from nanoquantization_b200.engine import LLMEngine
    from nanoquantization_b200.models.qwen3_quantized import Qwen3QuantizedForCausalLM
    make = lambda dim, dtype: Qwen3QuantizedForCausalLM(1, 64, 256, 256 // dim, 1, 32, 128, 4, 128, dim, device="cpu", dtype=dtype)  # noqa: E731
    with pytest.raises(ValueError, match="heads of 128"):
        LLMEngine(make(64, torch.float16), num_blocks=2, block_size=16, kv_bits=4)
    with pytest.raises(ValueError, match="multiple of 16"):
        LLMEngine(make(128, torch.float16), num_blocks=2, block_size=8, kv_bits=4)
    with pytest.raises(ValueError, match="4 or 16 bits"):
        LLMEngine(make(128, torch.float16), num_blocks=2, block_size=16, kv_bits=8)
    engine = LLMEngine(make(128, torch.bfloat16), num_blocks=2, block_size=16, max_batch=2, kv_bits=4)
    assert engine.cache.bits == 4 and engine.cache.k[0].shape == (3, 1, 16 * 72) and engine.cache.k[0].dtype == torch.uint8


def test_a_fork_holds_what_its_sequence_holds():
    from nanoquantization_b200.engine import LLMEngine, Sequence
    from nanoquantization_b200.models.qwen3_quantized import Qwen3QuantizedForCausalLM
    model = Qwen3QuantizedForCausalLM(1, 64, 256, 2, 1, 32, 128, 4, 128, 128, device="cpu", dtype=torch.float16)
    engine = LLMEngine(model, num_blocks=6, block_size=4, max_batch=2, use_cuda_graph=False)
    s = Sequence(3, [5, 6, 7, 8, 9, 10], 4, [11])
    assert engine.blocks.ensure(s, 7)
    s.computed = 6
    for c in (engine.cache.k[0], engine.cache.v[0]):
        c.copy_(torch.randn(c.shape))
    t = engine.fork(s)
    assert (t.prompt, t.output, t.blocks, t.computed, t.max_new_tokens) == (s.prompt, s.output, s.blocks, 6, 4) and t.prompt is not s.prompt
    before = engine.cache.k[0].clone()
    engine._hold(t, 8)
    assert t.blocks[0] == s.blocks[0] and t.blocks[1] != s.blocks[1]
    engine.blocks.flush()
    assert torch.equal(engine.cache.k[0][t.blocks[1]], before[s.blocks[1]])
    engine.drop(s), engine.drop(t)
    assert sorted(engine.blocks.free) == list(range(6))


def test_an_engine_goes_with_its_last_user():
    """No cycle of references: an engine that garbage collection took in the middle of another's graph capture would end that capture."""
    import gc
    import weakref
    from nanoquantization_b200.engine import LLMEngine
    from nanoquantization_b200.models.qwen3_quantized import Qwen3QuantizedForCausalLM
    model = Qwen3QuantizedForCausalLM(1, 64, 256, 2, 1, 32, 128, 4, 128, 128, device="cpu", dtype=torch.float16)
    gc.disable()
    try:
        for bits in (16, 4):
            engine = LLMEngine(model, num_blocks=2, block_size=16, max_batch=2, kv_bits=bits)
            gone = weakref.ref(engine)
            del engine
            assert gone() is None
    finally:
        gc.enable()


@pytest.mark.parametrize("seed", range(6))
def test_blocks_hold_what_their_sequences_wrote(seed):
    """Random growth, forks, copies, reclaims and releases over a pool whose contents are tracked."""
    import random
    from nanoquantization_b200.engine import BlockManager, Sequence
    rng, size, total = random.Random(seed), 4, 24
    m = BlockManager(total, size)
    memory = [[None] * size for _ in range(total)]

    def copy(pairs):
        assert len({b for _, b in pairs}) == len(pairs) and {a for a, _ in pairs}.isdisjoint(b for _, b in pairs)      # as copy_pages asks
        before = [list(x) for x in memory]
        for a, b in pairs:
            memory[b] = before[a]
    m.copy = copy
    live, next_id = [], 0

    def holders(b):
        return sum(b in s.blocks for s in live)
    for _ in range(600):
        what = rng.random()
        if what < 0.15 or not live:
            live.append(Sequence(next_id, [], 1 << 30))
            next_id += 1
        elif what < 0.3:
            s = rng.choice(live)
            t = Sequence(next_id, list(s.prompt), 1 << 30)
            t.computed = s.computed
            next_id += 1
            m.share(s, t)
            live.append(t)
        elif what < 0.4:
            s = live.pop(rng.randrange(len(live)))
            m.release(s)
        elif what < 0.45:
            s = rng.choice(live)
            s.first = max(getattr(s, "first", 0), rng.randint(0, s.computed) // size * size)
            m.reclaim(s, s.first)
        else:      # a step of one or several sequences, each with its next tokens
            step = []
            for s in rng.sample(live, rng.randint(1, len(live))):
                n = rng.choice([1, 1, 2, 5])
                if m.ensure(s, s.computed + n + rng.choice([0, 1])):
                    step.append((s, n))
            m.flush()
            for s, n in step:
                for _ in range(n):
                    s.prompt.append((s.seq_id, rng.random()))
                    block = s.blocks[s.computed // size]
                    assert block >= 0 and holders(block) == 1
                    memory[block][s.computed % size] = s.prompt[-1]
                    s.computed += 1
        if not m.copies:
            for s in live:
                for p in range(s.computed):
                    b = s.blocks[p // size]
                    assert b < 0 or memory[b][p % size] == s.prompt[p]
        used = {b for s in live for b in s.blocks if b >= 0}
        assert used.isdisjoint(m.free) and len(used) + len(m.free) == total and len(set(m.free)) == len(m.free)
        assert all(holders(b) == n + 1 for b, n in m.shared.items()) and all(holders(b) == 1 for b in used if b not in m.shared)
    for s in live:
        m.release(s)
    assert sorted(m.free) == list(range(total)) and not m.shared
