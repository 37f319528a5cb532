"""The 4-bit cache without a GPU: its format's bounds, what a part's cache need takes, options and refusals."""

import numpy as np
import pytest
import torch

import plain_q4 as q4
from conftest import TINY


def test_every_value_is_off_by_half_a_step_at_most():
    rng = np.random.default_rng(1)
    for scale in (1e-4, 0.02, 1.0, 300.0, 7e3):
        x = (rng.standard_normal((500, 64)) * scale).astype(np.float32)
        x[np.abs(x) > 57600] = 0
        n, s = q4.quantise(x)
        back = q4.values(n, s)
        step = np.repeat(np.array([q4.step_of(b) for b in s.reshape(-1)]).reshape(s.shape), 16, -1)
        # x * (1 / s) is rounded twice to 32 bits before rint: 2^-23 of at most 7.5
        assert (np.abs(back - x) <= step * (0.5 + 7.5 * 2.0 ** -22)).all()


def test_values_are_exact_in_bfloat16_and_steps_cover_the_range():
    assert q4.STEPS[1] == 2.0 ** -17 and q4.STEPS[-1] == 7680.0 and (np.diff(q4.STEPS) > 0).all()
    n, s = np.meshgrid(np.arange(1, 16), np.arange(q4.TOP + 1), indexing="ij")
    v = torch.from_numpy(q4.values(np.repeat(n.reshape(-1, 1), 16, 1), s.reshape(-1, 1)))
    assert torch.equal(v.to(torch.bfloat16).double(), v) and torch.equal(v.float().double(), v)


def test_needs_of_quantised_rows():
    from axon_b200.cache.manager import bytes_per_token
    from axon_b200.parts.spec import KvNeed
    for ps, hd, vd, planes in ((16, 128, 128, 2), (4, 64, 64, 2), (1, 16, 16, 2), (5, 48, 32, 2), (7, 32, 32, 1)):
        need = KvNeed(3, hd, v_dim=vd, planes=planes, bits=4)
        assert need.page_bytes(ps, 2) == 3 * q4.parts(ps, hd, vd, planes)[1]
    assert bytes_per_token([KvNeed(4, 128, bits=4)], torch.bfloat16) == 4 * 2 * 72
    assert bytes_per_token([KvNeed(4, 128)], torch.bfloat16) == 4 * 2 * 256
    assert bytes_per_token([KvNeed(1, 16, bits=4)], torch.float32, 1) == 64      # four parts padded to 16 bytes
    with pytest.raises(ValueError, match="multiple of 16"):
        KvNeed(2, 24, bits=4)
    with pytest.raises(ValueError, match="multiple of 16"):
        KvNeed(2, 32, v_dim=40, bits=4)
    with pytest.raises(ValueError, match="not 8"):
        KvNeed(2, 32, bits=8)


def test_only_parts_that_take_it_keep_a_quantised_cache():
    from axon_b200.config import config_from_dict
    from axon_b200.config.base import architecture_of
    from axon_b200.engine.model import layer_cache_needs
    cfg = config_from_dict(TINY["A"])
    spec = architecture_of(cfg.to_dict()).build_spec(cfg)
    assert [n.bits for n in layer_cache_needs(spec.layers[0]).values()] == [0]
    assert [n.bits for n in layer_cache_needs(spec.layers[0], 4).values()] == [4]
    from axon_b200.parts.base import Mixer, Runtime
    assert Mixer.kv_bits == ()
    with pytest.raises(ValueError, match="4 bits"):
        Runtime(torch.bfloat16, "cpu", kv_bits=8)


def test_cache_types_by_name():
    from axon_b200.api import BackendOptions
    from axon_b200.engine.build import parse_kv
    assert BackendOptions().kv("q4")._kv == "q4" and BackendOptions().kv("bf16")._kv == "auto"
    assert BackendOptions().kv("q4").kv("auto")._kv == "auto"
    assert parse_kv("q4", "float32") == 4 and parse_kv("auto", torch.bfloat16) == 0
    with pytest.raises(ValueError, match="q8"):
        BackendOptions().kv("q8")
    with pytest.raises(ValueError, match="differs"):
        BackendOptions().kv("f32")


def test_which_segments_are_read_back():
    """The rule between the 4-bit kernel and reading back, against measured times (microseconds: 4-bit kernel, read back)."""
    from types import SimpleNamespace
    from axon_b200.kernels import fast
    measured = {  # (heads, kv heads, head size, requests, tokens, positions)
        (28, 4, 128, 1, 16, 8192): (25, 154), (28, 4, 128, 1, 128, 8192): (81, 183), (28, 4, 128, 1, 128, 1024): (24, 34),
        (28, 4, 128, 8, 32, 2048): (54, 63), (28, 4, 128, 8, 64, 2048): (94, 64), (28, 4, 128, 1, 128, 32768): (273, 702),
        (28, 4, 128, 1, 2048, 8192): (892, 331), (12, 2, 128, 8, 64, 2048): (49, 58), (12, 2, 128, 1, 128, 32768): (125, 695),
        (14, 2, 64, 8, 64, 2048): (35, 71), (14, 2, 64, 1, 128, 8192): (28, 251),
    }
    for (heads, kv_heads, hd, n, tokens, kv), (short, long) in measured.items():
        ctx = SimpleNamespace(seg_q_len=[tokens] * n, seg_kv_len=[kv] * n, max_q_len=tokens, scratch={})
        took = fast._q4_long(ctx, heads // kv_heads, kv_heads, hd, 0, True)
        assert len(took) in (0, n) and (bool(took) == (long < short)), (heads, kv_heads, hd, n, tokens, kv)
    mixed = SimpleNamespace(seg_q_len=[1, 2000, 9, 1900], seg_kv_len=[5000, 2000, 40, 1900], max_q_len=2000, scratch={})
    assert fast._q4_long(mixed, 7, 4, 128, 0, True) == (1, 3)
    assert fast._q4_long(mixed, 2, 1, 16, 0, False) == (0, 1, 2, 3)       # no 4-bit kernel: everything, once something is long
    assert fast._q4_long(mixed, 7, 4, 256, 0, True) == ()
    few = SimpleNamespace(seg_q_len=[1, 3], seg_kv_len=[5000, 2000], max_q_len=3, scratch={})
    assert fast._q4_long(few, 2, 1, 16, 0, False) == () and not few.scratch


def test_room_for_prompts_is_never_outgrown():
    """What a step's prompts need, however they lie, fits the buffers that the engine asks for once."""
    from types import SimpleNamespace
    from axon_b200.engine.build import quantised_workspace_bytes
    from axon_b200.kernels import fast
    from axon_b200.parts.spec import KvNeed
    rng = np.random.default_rng(5)
    for slots, most, pool in ((1, 100, 128), (16, 4096, 65536), (8, 32768, 100000), (128, 2000, 20000), (300, 70, 21000)):
        pages, ints = fast.q4_prompt_room(slots, most, pool)
        for _ in range(30):
            n = int(rng.integers(1, slots + 1))
            kv = np.minimum(rng.integers(1, most + 1, n), max(1, pool // n))
            q = np.minimum(rng.integers(1, most + 1, n), kv)
            if kv.sum() > max(most, fast.Q4_PROMPT_POSITIONS):
                continue                                  # (such a step is taken in groups)
            ctx = SimpleNamespace(seg_q_len=q.tolist(), seg_kv_len=kv.tolist())
            for window in (0, 50):
                p, stride = fast._q4_prompt_sizes(ctx, range(n), window)
                assert p <= pages and 8 * n + n * stride <= ints
    assert quantised_workspace_bytes([{"mixer": KvNeed(4, 128)}], 16, 4096) == 0
    assert quantised_workspace_bytes([{"mixer": KvNeed(4, 128, bits=4)}, {}], 16, 4096) >= 65536 * 4 * 2 * 128 * 2


def test_views_of_quantised_pools_are_checked():
    from axon_b200.kernels import ops
    table = torch.zeros(1, 4, dtype=torch.int32)
    good = torch.zeros(5, 2, 2 * (q4.parts(16, 64, 64, 2)[1]), dtype=torch.uint8)
    view = ops.KvView(good, table, 1, 16, 2, 64, bits=4)
    assert view.layout.bits == 4 and view.layout.entry_offset == good.shape[2] and view.n_pages == 4
    with pytest.raises(ValueError, match="kv_read"):
        view.keys()
    with pytest.raises(ValueError, match="uint8"):
        ops.KvView(good.to(torch.int8), table, 1, 16, 2, 64, bits=4)
    with pytest.raises(ValueError, match="does not hold"):
        ops.KvView(good[:, :, 16:].contiguous(), table, 1, 16, 2, 64, bits=4)
    with pytest.raises(ValueError, match="int32"):
        ops.KvView(good, table.long(), 1, 16, 2, 64, bits=4)
    with pytest.raises(ValueError, match="multiple of 16"):
        ops.KvView(good, table, 1, 16, 2, 40, bits=4)


def division(tiles, kv_heads, ctas):
    """How an attention launch divides items of these many tiles: (places in all, of a CTA, before a pair, padded)."""
    from axon_b200.kernels import lib
    t, out = np.ascontiguousarray(tiles, np.int32), np.zeros(4, np.uint32)
    lib.check(lib.cuda().axon_attention_q4_division(t.ctypes.data, len(t), kv_heads, ctas, out.ctypes.data))
    return [int(x) for x in out]


def check_division(tiles, kv_heads, ctas):
    """Every pair's tiles lie in the ranges that the CTAs go through, worked out in unbounded integers."""
    total, per, cost, padded = division(tiles, kv_heads, ctas)
    tiles = np.asarray(tiles, np.int64)
    weights = np.where(tiles == 0, 0, -(-tiles // per) * per if padded else tiles + cost)
    assert total == int(weights.sum()) * kv_heads < 2 ** 32, "the places of all pairs were miscounted"
    assert total <= ctas * per < 2 ** 32, "there are more places than the CTAs go through"
    assert per >= 8 and (not padded or per % 8 == 0)
    # a CTA has two pieces of others' pairs at most: where pairs follow one another, those that its range begins and ends in
    if padded:
        assert cost == 0 and int((-(-tiles // per)).sum()) * kv_heads <= ctas
    return padded


def test_work_is_divided_whole():
    """The guard of the launcher lets through up to 2**31 tiles with what pairs cost; the division counts them all."""
    rng = np.random.default_rng(8)
    seen = set()
    for k in range(400):
        kv_heads, ctas = int(rng.choice([1, 2, 4, 8, 16])), int(rng.choice([148, 296]))
        n = int(np.exp(rng.uniform(0, np.log(33000))))
        most = 2 ** 31 // (n * kv_heads) - 25
        longest = int(np.exp(rng.uniform(0, np.log(max(min(most, 2 ** 27), 2)))))
        kind = k % 4
        tiles = (np.full(n, longest) if kind == 0 else rng.integers(0, longest + 1, n) if kind == 1 else
                 np.maximum(longest - np.arange(n) // 2, 1) if kind == 2 else np.where(rng.random(n) < 0.02, longest, rng.integers(0, 9, n)))
        if tiles.sum() == 0:
            continue
        seen.add(check_division(tiles, kv_heads, ctas))
    assert seen == {0, 1}
    for n, kv_heads in ((1, 1), (148, 1), (149, 1), (33000, 8)):        # the largest that the launcher takes
        check_division(np.full(n, 2 ** 31 // (n * kv_heads) - 25), kv_heads, 148)


# heads, kv heads of 256, tokens, positions at the portion's end: pairs times the longest range pass 2**32 and wrap to a small number
PORTIONS_THAT_WRAP = [(32, 8, 4096, 39936), (32, 8, 4096, 77824), (32, 8, 4096, 115712), (16, 8, 8192, 41984), (16, 16, 8192, 41984), (64, 8, 2048, 38912)]


@pytest.mark.parametrize("heads,kv_heads,tokens,end", PORTIONS_THAT_WRAP)
def test_portions_of_very_many_items_are_divided_whole(heads, kv_heads, tokens, end):
    group = heads // kv_heads
    rows = np.arange(0, tokens * group, 8)
    tiles = (end - tokens + np.minimum(tokens, -(-(rows + 8) // group)) + 15) // 16
    assert not check_division(tiles, kv_heads, 148)


def test_key_shares_of_the_plain_attention():
    """Few different counts while a context grows (each is a captured step), no share of more than 64 keys unless the GPU is full,
    and scratch whose size follows none of it."""
    from types import SimpleNamespace
    from axon_b200.kernels import fast, lib
    for heads, kv_heads, tokens, window in ((8, 2, 1, 0), (6, 1, 1, 0), (28, 4, 3, 0), (8, 2, 4, 1024), (8, 8, 64, 0), (40, 2, 1, 0)):
        counts = set()
        for kv in range(1, 30000, 7):
            ctx = SimpleNamespace(max_kv_len=kv, n_tokens=tokens)
            n = fast.q4_plain_splits(ctx, heads, kv_heads, window)
            tiles = -(-(min(kv, window) if window else kv) // 64)
            full = max(1, fast.Q4_PLAIN_CTAS // (tokens * kv_heads * -(-(heads // kv_heads) // 8)))
            assert n >= min(tiles, full) and n <= max(full, 1) and (n <= tiles * 1.25 or n == 1)
            counts.add(n)
            if n > 1:
                assert lib.cuda().axon_attention_q4_plain_scratch(tokens, heads, kv_heads, 64, n) <= fast.Q4_PLAIN_CTAS * fast.Q4_PLAIN_HEADS * 66
                assert tokens * kv_heads * -(-(heads // kv_heads) // 8) <= fast.Q4_PLAIN_CTAS
        assert len(counts) <= 36, len(counts)


def test_memory_that_prompts_are_read_back_into():
    """Counted for each count and size of heads that can be read back, not at all for the 32-bit model."""
    from axon_b200.engine.build import quantised_workspace_bytes
    from axon_b200.kernels import fast
    from axon_b200.parts.spec import KvNeed, StateNeed
    a, b = KvNeed(4, 128, bits=4), KvNeed(2, 64, window=100, bits=4)
    needs = [{"x": a}, {"x": b, "y": StateNeed((3,), "float32")}, {"x": KvNeed(4, 128, window=50, bits=4)}, {}, {"x": KvNeed(8, 128)},
             {"x": KvNeed(1, 256, bits=4)}, {"x": KvNeed(1, 64, v_dim=32, bits=4)}, {"x": KvNeed(1, 64, planes=1, bits=4)}]
    pages, ints = fast.q4_prompt_room(16, 4096, 65536)
    assert fast.q4_prompt_buffers(needs, pages) == {fast._q4_pages_name(4, 128): (pages, 2, 4, 64, 128), fast._q4_pages_name(2, 64): (pages, 2, 2, 64, 64)}
    each = [quantised_workspace_bytes([{"x": n}], 16, 4096) for n in (a, b)]
    assert each[0] == pages * 64 * 2 * 4 * 128 * 2 + 4 * ints and quantised_workspace_bytes(needs, 16, 4096) == sum(each)
    assert quantised_workspace_bytes(needs, 16, 4096, torch.float32) == 0
    assert quantised_workspace_bytes([{"x": KvNeed(1, 256, bits=4)}], 16, 4096) == 0


def test_an_attention_that_keeps_the_models_dtype_keys_its_steps_by_its_split_count():
    """A part that does not take the 4-bit format launches the kernels of whole elements beside parts that do."""
    from types import SimpleNamespace
    from axon_b200.parts.standard import Attention

    class Whole(Attention):
        kv_bits = ()

    keys = {}
    for cls in (Attention, Whole):
        part = object.__new__(cls)
        part.rt = SimpleNamespace(kv_bits=4, precise=False, kv_page_size=16)
        part.heads, part.kv_heads, part.head_dim, part.window = 28, 4, 128, 0
        for kv in (100, 30000):
            ctx = SimpleNamespace(rt=part.rt, seg_q_len=[1], seg_kv_len=[kv], n_tokens=1, max_q_len=1, max_kv_len=kv, scratch={})
            keys[cls, kv] = part.graph_key(ctx)
    assert keys[Attention, 100] == keys[Attention, 30000] == ()
    assert keys[Whole, 100] != keys[Whole, 30000]
