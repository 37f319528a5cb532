"""The 4-bit cache's operators on the GPU against ``plain_q4``: rotating and quantising rows as they are
written, reading them back, attention over the pages, and the engine with such a cache."""

import math

import numpy as np
import pytest
import torch

import plain_q4 as q4

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16]
#: half a step of a rounding to each type, relative to the value
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def ops():
    from axon_b200.kernels import ops as o
    return o


class Cache:
    """Requests of given lengths in a pool whose other bytes are all 0xFF (steps that read as NaN)."""

    def __init__(self, ops, lens, kv_heads, hd, ps, v_dim=None, planes=2, window=0, seed=0, room=0, fill=True, spare=3, loud=0.0):
        self.lens, self.kv_heads, self.hd, self.ps, self.planes = lens, kv_heads, hd, ps, planes
        self.v_dim = hd if v_dim is None or planes == 1 else v_dim
        rng = np.random.default_rng(seed)
        stride = -(-(max(lens) + room) // ps)
        held = [-(-(l + room) // ps) for l in lens]
        n_pages = sum(held) + spare
        order = rng.permutation(n_pages)
        self.table = np.full((len(lens), stride), n_pages, np.int32)
        at = 0
        for i, n in enumerate(held):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.places, self.record = q4.parts(ps, hd, self.v_dim, planes)
        pool = np.full((n_pages + 1, 2, kv_heads * self.record), 0xFF, np.uint8)
        shift = rng.standard_normal((kv_heads, hd)) * loud
        self.k = [(rng.standard_normal((l, kv_heads, hd)) + shift).astype(np.float32) for l in lens]
        self.v = [rng.standard_normal((l, kv_heads, self.v_dim)).astype(np.float32) for l in lens]
        if fill:
            for s, l in enumerate(lens):
                rows = [q4.quantise(self.k[s])] + ([q4.quantise(self.v[s])] if planes == 2 else [])
                self.k[s] = q4.values(*rows[0])
                self.v[s] = q4.values(*rows[-1])
                for p in range(l):
                    for h in range(kv_heads):
                        for j, (n, b) in enumerate(rows):
                            page = int(self.table[s, p // ps])
                            q4.put(pool, page, 1, h, self.record, self.places[2 * j], p % ps, q4.codes_of(n[p, h]))
                            q4.put(pool, page, 1, h, self.record, self.places[2 * j + 1], p % ps, b[p, h])
        self.pool = torch.from_numpy(pool).to(DEV)
        self.dev_table = torch.from_numpy(self.table).to(DEV)
        self.view = ops.KvView(self.pool, self.dev_table, 1, ps, kv_heads, hd, window, v_dim=self.v_dim, planes=planes, bits=4)


def rotated(x, table, rot, adjacent):
    """Rows [n, heads, hd] of float32, every product and sum rounded to 32 bits."""
    x = x.copy()
    if not rot:
        return x
    c, s = table[:, None, :, 0], table[:, None, :, 1]
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if adjacent else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., first].copy(), x[..., second].copy()
    x[..., first], x[..., second] = a * c - b * s, a * s + b * c
    return x


def rope(positions, rot, theta=1e4):
    inv = theta ** (-2.0 * np.arange(rot // 2) / rot)
    ang = np.asarray(positions, np.float64)[:, None] * inv[None]
    return np.stack((np.cos(ang), np.sin(ang)), -1).astype(np.float32)


def i32(x):
    return torch.tensor(np.asarray(x, np.int32), device=DEV)


WRITES = [  # heads, kv heads, head size, rot, adjacent, page size, v_dim, planes
    (4, 2, 16, 16, False, 4, None, 2), (3, 1, 32, 32, True, 16, None, 2), (5, 5, 48, 16, False, 5, None, 2),
    (7, 1, 128, 128, False, 16, None, 2), (2, 2, 64, 0, False, 1, None, 2), (4, 2, 64, 12, False, 16, None, 2),
    (4, 2, 64, 10, True, 8, None, 2), (2, 1, 256, 256, False, 16, None, 2), (2, 2, 32, 32, False, 7, 48, 2),
    (4, 1, 64, 64, False, 16, None, 1),
]


def write_case(ops, dtype, heads, kv_heads, hd, rot, adjacent, ps, v_dim, planes, qkv, positions, slots, pending=None, write_kv=True,
               qkv_dev=None):
    """Runs rope_kv_write on an empty cache of two requests; the cache, q and the pool it must have left."""
    cache = Cache(ops, [40, 23], kv_heads, hd, ps, v_dim, planes, fill=False)
    want = cache.pool.cpu().numpy().copy()
    n = len(positions)
    tab = rope(positions, rot) if rot else None
    q = torch.full((n, heads * hd), 7.0, dtype=dtype, device=DEV)
    ops.rope_kv_write(qkv_dev if qkv_dev is not None else torch.from_numpy(qkv).to(DEV), None if tab is None else torch.from_numpy(tab).to(DEV),
                      i32(positions), i32(slots), q, cache.view, heads, rot, adjacent, write_kv=write_kv, pending=pending)
    qd, kd = heads * hd, kv_heads * hd
    x = rotated(qkv[:, :qd + kd].reshape(n, heads + kv_heads, hd), tab, rot, adjacent)
    k, v = x[:, heads:], qkv[:, qd + kd:].reshape(n, -1, cache.v_dim) if planes == 2 else None
    if write_kv:
        for t in range(n):
            for h in range(kv_heads):
                q4.store_row(want, cache.table, slots[t], positions[t], 1, h, ps, hd, cache.v_dim, planes, k[t, h], None if v is None else v[t, h])
    return cache, q, x[:, :heads].reshape(n, -1), want


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,hd,rot,adjacent,ps,v_dim,planes", WRITES)
def test_write(ops, dtype, heads, kv_heads, hd, rot, adjacent, ps, v_dim, planes):
    positions, slots = [0, 1, 2, 3, 4, 5, 16, 39, 0, 21, 22], [0] * 8 + [1] * 3
    width = (heads + kv_heads) * hd + (kv_heads * (v_dim or hd) if planes == 2 else 0)
    qkv = (np.random.default_rng(3).standard_normal((len(positions), width)) * 2).astype(np.float32)
    cache, q, want_q, want = write_case(ops, dtype, heads, kv_heads, hd, rot, adjacent, ps, v_dim, planes, qkv, positions, slots)
    got = cache.pool.cpu().numpy()
    assert (got == want).all(), f"{(got != want).sum()} bytes of the pool differ"
    err = np.abs(q.double().cpu().numpy() - want_q.astype(np.float64))
    assert (err <= HALF[dtype] * np.abs(want_q) + 1e-45).all()      # q is rounded once from the same 32-bit numbers
    cache, q, _, want = write_case(ops, dtype, heads, kv_heads, hd, rot, adjacent, ps, v_dim, planes, qkv, positions, slots, write_kv=False)
    assert (cache.pool.cpu().numpy() == 0xFF).all()


def test_write_of_numbers_that_quantise_badly(ops):
    """Groups of zeros, of subnormals, below the smallest step, at its border, over the largest, not finite."""
    rows = np.zeros((12, 48), np.float32)
    rows[1] = 1e-42
    rows[2] = 3.0e-6                              # less than half the smallest step: zero
    rows[3] = 4.0e-6
    rows[4, 5], rows[4, 20], rows[4, 40] = np.inf, np.nan, -np.inf
    rows[4, 6] = 1.0
    rows[5] = 6e4                                 # saturates
    rows[6] = -3e38
    rows[7] = np.float32(2.0 ** -14 * 7.5)        # where subnormal steps end
    rows[8] = np.nextafter(np.float32(2.0 ** -14 * 7.5), np.float32(1))
    rows[9] = np.repeat([7.5, 15.0, 60.0], 16)    # the step is a power of two, the largest exactly 7.5 steps: held as 7
    rows[10] = np.tile([0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 7.0, 7.5], 6)   # halves of a step: to even
    rows[11, ::16], rows[11, 1::16] = 1e-3, -0.0
    qkv = np.concatenate([np.ones((12, 48), np.float32), rows, rows[::-1]], 1)
    positions = list(range(12))
    cache, _, _, want = write_case(ops, torch.float32, 1, 1, 48, 0, False, 16, None, 2, qkv, positions, [0] * 12)
    assert (cache.pool.cpu().numpy() == want).all()
    keys = torch.empty(12, 1, 48, device=DEV)
    ops.kv_read(cache.view, i32([[0], [0], [12], [0]]), keys)
    got = keys[:, 0].double().cpu().numpy()
    assert np.isnan(got[4]).all() and (got[:3] == 0).all() and (got[5] == 53760).all() and (got[6] == -53760).all()
    assert (got[10, :8] == [0, 2, 2, 0, -2, -2, 7, 7]).all()


@pytest.mark.parametrize("splits", [1, 3, 9])
@pytest.mark.parametrize("hd,rot", [(64, 64), (48, 12)])
def test_write_folds_partial_sums(ops, splits, hd, rot):
    """The q/k/v product may still lie in scratch as partial sums (slabs of 128 columns)."""
    from axon_b200.kernels import fast
    heads, kv_heads, n, ntok = 4, 2, 5, 16
    width = (heads + 2 * kv_heads) * hd
    cols = -(-width // 128)
    rng = np.random.default_rng(5)
    part = rng.standard_normal((cols, splits, ntok, 128)).astype(np.float32)
    bias = rng.standard_normal(width).astype(np.float32)
    full = np.zeros((n, cols * 128), np.float32)
    for s in range(splits):
        full += part[:, s, :n].transpose(1, 0, 2).reshape(n, -1)
    qkv = full[:, :width] + bias
    out = torch.zeros(n, width, device=DEV)
    owed = fast.PendingFold(torch.from_numpy(part).to(DEV), splits, ntok, torch.from_numpy(bias).to(DEV), out, False)
    cache, _, _, want = write_case(ops, torch.bfloat16, heads, kv_heads, hd, rot, False, 16, None, 2, qkv, [0, 1, 2, 17, 39], [0] * 5,
                                   pending=owed, qkv_dev=out)
    assert owed.claimed and (cache.pool.cpu().numpy() == want).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv_heads,hd,ps,v_dim,planes", [(2, 16, 4, None, 2), (1, 64, 1, None, 2), (4, 128, 16, None, 2), (3, 48, 7, 32, 2),
                                                         (2, 32, 16, None, 1), (2, 256, 32, None, 2)])
def test_read(ops, dtype, kv_heads, hd, ps, v_dim, planes):
    cache = Cache(ops, [70, 1, 33], kv_heads, hd, ps, v_dim, planes, seed=4)
    # parts of requests in no order, an empty one, rows between them that belong to none, two rows asked for twice
    spans = [(2, 5, 28, 0), (0, 0, 70, 30), (1, 0, 1, 101), (0, 3, 0, 103), (2, 32, 1, 104), (0, 60, 4, 98)]
    rows = 110
    keys = torch.full((rows, kv_heads, hd), -5.0, dtype=dtype, device=DEV)
    vals = torch.full((rows, kv_heads, cache.v_dim), -5.0, dtype=dtype, device=DEV)
    ops.kv_read(cache.view, i32(spans).T.contiguous(), keys, vals)
    want_k, want_v = np.full(keys.shape, -5.0), np.full(vals.shape, -5.0)
    for slot, first, count, out in reversed(spans):
        want_k[out:out + count], want_v[out:out + count] = cache.k[slot][first:first + count], cache.v[slot][first:first + count]
    assert (keys.double().cpu().numpy() == want_k).all() and (vals.double().cpu().numpy() == want_v).all()
    only = torch.full_like(vals, -5.0)
    ops.kv_read(cache.view, i32(spans).T.contiguous(), None, only)
    assert torch.equal(only, vals)


def test_read_leaves_what_lies_outside_the_table(ops):
    cache = Cache(ops, [20, 9], 2, 64, 16, seed=6)
    keys = torch.full((40, 2, 64), -5.0, device=DEV)
    # a slot too many, a negative one, a negative position, positions past the table's end
    ops.kv_read(cache.view, i32([[2, -1, 0, 0], [0, 0, -3, 18], [5, 5, 5, 20], [0, 5, 10, 15]]), keys)
    got = keys.double().cpu().numpy()
    assert (got[:13] == -5).all() and (got[13:15] == cache.k[0][:2]).all() and (got[15:17] == cache.k[0][18:20]).all()
    assert (got[15 + 14:] == -5).all(), "positions beyond the block table were read"


def test_refusals(ops):
    from axon_b200.kernels.lib import KernelError
    cache = Cache(ops, [20], 2, 64, 16)
    keys, spans = torch.zeros(4, 2, 64, device=DEV), i32([[0], [0], [4], [0]])
    for bad, what in (((spans.long(), keys), "int32 spans"), ((spans[:3].contiguous(), keys), "spans"), ((spans, keys[:, :1].contiguous()), "keys as"),
                      ((spans, None), "both"), ((spans, keys, torch.zeros(3, 2, 64, device=DEV)), "values as")):
        with pytest.raises(ValueError, match=what):
            ops.kv_read(cache.view, *bad)
    with pytest.raises(TypeError, match="one dtype"):
        ops.kv_read(cache.view, spans, keys, keys.to(torch.bfloat16))
    with pytest.raises(TypeError, match="float16"):
        ops.kv_read(cache.view, spans, keys.half())
    with pytest.raises(ValueError, match="contiguous CUDA"):
        ops.kv_read(cache.view, spans, torch.zeros(4, 2, 128, device=DEV)[..., :64])
    plain = ops.KvView(torch.zeros(3, 1, 2, 2, 16, 64, device=DEV), cache.dev_table, 0, 16, 2, 64)
    with pytest.raises(ValueError, match="quantised rows"):
        ops.kv_read(plain, spans, keys)
    qkv, pos = torch.zeros(4, 8 * 64, device=DEV), i32([0, 1, 2, 3])
    q = torch.zeros(4, 4 * 64, device=DEV)
    with pytest.raises(ValueError, match="for each row"):
        ops.rope_kv_write(qkv, None, pos[:3].contiguous(), pos, q, cache.view, 4, 0)
    with pytest.raises(ValueError, match="for each row"):
        ops.rope_kv_write(qkv, None, pos, pos, q[:, :64].contiguous(), cache.view, 4, 0)
    with pytest.raises(TypeError, match="int32"):
        ops.rope_kv_write(qkv, None, pos.long(), pos, q, cache.view, 4, 0)
    with pytest.raises(TypeError, match="float16"):
        ops.rope_kv_write(qkv, None, pos, pos, q.half(), cache.view, 4, 0)
    with pytest.raises(ValueError, match="rotation table"):
        ops.rope_kv_write(qkv, torch.zeros(4, 16, 2, device=DEV), pos, pos, q, cache.view, 4, 64)
    with pytest.raises(KernelError, match="rotated size"):
        ops.rope_kv_write(qkv, torch.zeros(4, 64, 2, device=DEV), pos, pos, q, cache.view, 4, 128)
    with pytest.raises(ValueError, match="queries"):
        ops.attention_plain(q, cache.view, pos, pos, q[:, :64].contiguous(), 4, 0.1)
    with pytest.raises(KernelError, match="over 2 kv heads"):
        ops.attention_plain(torch.zeros(4, 3 * 64, device=DEV), cache.view, pos, pos, torch.zeros(4, 3 * 64, device=DEV), 3, 0.1)


def test_other_launchers_refuse_quantised_pools(ops):
    """The kernels of caches in whole elements look at the layout, whoever calls them."""
    from axon_b200.kernels import lib
    cache = Cache(ops, [20], 2, 64, 16)
    x, one = torch.zeros(1, 4 * 64, dtype=torch.bfloat16, device=DEV), i32([0, 0, 1, 1])
    calls = {
        "axon_rope_kv_write": (torch.zeros(1, 8 * 64, device=DEV).data_ptr(), None, one.data_ptr(), one.data_ptr(), x.data_ptr(),
                               cache.pool.data_ptr(), 1, cache.view._ref, 1, 4, 0, 0, 1, None, 0, 0, None, lib.current_stream()),
        "axon_attention_plain": (x.data_ptr(), cache.pool.data_ptr(), 1, one.data_ptr(), one.data_ptr(), x.data_ptr(), cache.view._ref, 1, 4,
                                 0.1, 0, lib.current_stream()),
        "axon_attention_fa": (x.data_ptr(), cache.pool.data_ptr(), x.data_ptr(), one.data_ptr(), 1, None, 1, cache.view._ref, 4, 0.1, 0, 1, 1, 1,
                              None, None, lib.current_stream()),
        "axon_attention_tc": (x.data_ptr(), cache.pool.data_ptr(), x.data_ptr(), one.data_ptr(), 1, one.data_ptr(), 1, cache.view._ref, 4, 0.1, 0,
                              1, lib.current_stream()),
    }
    for name, args in calls.items():
        with pytest.raises(lib.KernelError, match="4 bits"):
            lib.check(getattr(lib.cuda(), name)(*args))


# -- attention --------------------------------------------------------------

def attend(ops, cache, q_lens, heads, dtype, window=0, seed=9, scale=None, rt=None, precise=None, q=None):
    """linear.attention for the last ``q_lens[s]`` tokens of each request; (out, context, q)."""
    from axon_b200.kernels import linear
    from axon_b200.parts.base import Runtime, StepContext
    hd, vd = cache.hd, cache.v_dim
    n = sum(q_lens)
    if q is None:
        q = (torch.randn(n, heads * hd, generator=torch.Generator().manual_seed(seed)) * 1.5).to(dtype).to(DEV)
    starts = [sum(q_lens[:i]) for i in range(len(q_lens))]
    pos = [p for l, k in zip(cache.lens, q_lens) for p in range(l - k, l)]
    slot = [s for s, k in enumerate(q_lens) for _ in range(k)]
    live = [s for s, k in enumerate(q_lens) if k]
    seg = [live, [starts[s] for s in live], [q_lens[s] for s in live], [cache.lens[s] for s in live]]
    rt = rt or Runtime(dtype, DEV, kv_bits=4)
    ctx = StepContext(rt=rt, n_tokens=n, tokens=None, positions=i32(pos), token_slot=i32(slot), seg_slot=seg[0], seg_q_start=seg[1],
                      seg_q_len=seg[2], seg_kv_len=seg[3], segments=i32(seg),
                      unit_items=i32([[i, 0] for i in range(len(live))]) if all(k == 1 for k in seg[2]) else None)
    out = torch.full((n + 2, heads * vd), -7.0, dtype=dtype, device=DEV)
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    linear.attention(q, cache.view, ctx, out[:n], heads, scale, precise=dtype == torch.float32 if precise is None else precise)
    assert (out[n:] == -7.0).all(), "rows behind the last token were written"
    return out[:n], ctx, q, pos, slot, scale


def check_attention(ops, cache, q_lens, heads, dtype, window=0, weight_half=2.0 ** -11, **kw):
    """Against float64, within a bound worked out for each number: a score is a sum of hd products in
    32 bits (2^-23 a step: tensor cores cut sums), scaled (2^-22 of its size with the exponential's own error),
    a weight is rounded to half its step (``weight_half``; none in the 32-bit model), sums over keys and the
    output round again.

    Weights below 2^-14 of the running maximum's are subnormal halves in the kernel for few rows: off by 2^-25
    at most, whatever their size.  The running maximum never exceeds the row's, so the largest weight and the sum
    that all are divided by are at least 1, and the output is off by 2^-25 times the sum of |v| at most."""
    out, ctx, q, pos, slot, scale = attend(ops, cache, q_lens, heads, dtype, window, **kw)
    got = out.double().cpu().numpy().reshape(len(pos), heads, -1)
    qd = q.double().cpu().numpy().reshape(len(pos), heads, -1)
    group = heads // cache.kv_heads
    pos, slot = np.array(pos), np.array(slot)
    weight = 0.0 if dtype == torch.float32 else weight_half
    for s in set(slot.tolist()):
        rows = np.nonzero(slot == s)[0]
        for h in range(heads):
            want, mass, size = q4.attention(qd[rows, h], cache.k[s][:, h // group], cache.v[s][:, h // group], pos[rows], window, scale)
            e_s = size * ((cache.hd + 4) * 2.0 ** -23 + 2.0 ** -22)
            tiny = 2.0 ** -25 * np.abs(cache.v[s][:, h // group]).sum(0) if weight else 0.0
            tol = tiny + mass * (weight + 2 * e_s[:, None] + 2.0 ** -20 + (cache.lens[s] + 8) * 2.0 ** -23) + 1.01 * HALF[dtype] * np.abs(want) + 1e-30
            err = np.abs(got[rows, h] - want)
            assert (err <= tol).all(), f"request {s} head {h}: worst error {float((err / tol).max()):.2f} of its bound"
    return out, ctx


LAYOUTS = [  # heads, kv heads, head size, page size
    (4, 2, 16, 4), (3, 1, 32, 16), (5, 5, 48, 5), (2, 1, 256, 16), (28, 4, 128, 16), (12, 2, 128, 32), (6, 2, 64, 16), (8, 8, 128, 8),
    (9, 1, 64, 4), (20, 1, 128, 64), (40, 1, 128, 16), (6, 2, 128, 48), (4, 4, 64, 1),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,hd,ps", LAYOUTS)
@pytest.mark.parametrize("window", [0, 1, 37])
def test_single_tokens(ops, dtype, heads, kv_heads, hd, ps, window):
    cache = Cache(ops, [1, 2, 15, 16, 17, 33, 70, 130, 257], kv_heads, hd, ps, window=window, seed=11)
    check_attention(ops, cache, [1] * 9, heads, dtype, window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,hd,ps", LAYOUTS)
@pytest.mark.parametrize("window", [0, 19])
def test_portions(ops, dtype, heads, kv_heads, hd, ps, window):
    """Portions of one to a few dozen tokens beside requests that have none in this step."""
    cache = Cache(ops, [2, 40, 5, 64, 81, 33], kv_heads, hd, ps, window=window, seed=12)
    check_attention(ops, cache, [2, 3, 0, 9, 1, 33], heads, dtype, window, weight_half=2.0 ** -8)


@pytest.mark.parametrize("heads,kv_heads,hd,ps,lens", [(28, 4, 128, 16, [5003]), (12, 2, 128, 16, [4096, 1, 777]), (6, 2, 64, 32, [3000, 2999]),
                                                       (5, 5, 48, 16, [2500, 3])])
@pytest.mark.parametrize("window", [0, 1000])
def test_long_contexts_in_shares(ops, heads, kv_heads, hd, ps, lens, window):
    cache = Cache(ops, lens, kv_heads, hd, ps, window=window, seed=13, loud=1.0)
    check_attention(ops, cache, [1] * len(lens), heads, torch.bfloat16, window)
    check_attention(ops, cache, [min(l, 4) for l in lens], heads, torch.bfloat16, window, weight_half=2.0 ** -8)
    check_attention(ops, cache, [1] * len(lens), heads, torch.float32, window)


@pytest.mark.parametrize("heads,kv_heads,hd,ps", [(28, 4, 128, 16), (6, 2, 64, 32), (3, 1, 32, 16), (4, 2, 16, 5), (64, 1, 128, 16), (7, 1, 128, 7),
                                                  (4, 1, 256, 16), (65, 1, 64, 16)])
@pytest.mark.parametrize("window", [0, 100])
def test_prompts(ops, heads, kv_heads, hd, ps, window):
    """Prompts whole and at the end of longer requests, beside short portions and single tokens."""
    cache = Cache(ops, [300, 700, 41, 1, 650, 129], kv_heads, hd, ps, window=window, seed=21, loud=0.5)
    check_attention(ops, cache, [300, 259, 3, 1, 100, 0], heads, torch.bfloat16, window, weight_half=2.0 ** -8)
    check_attention(ops, cache, [0, 0, 0, 0, 0, 129], heads, torch.bfloat16, window, weight_half=2.0 ** -8)
    check_attention(ops, cache, [0, 700, 0, 0, 650, 0], heads, torch.bfloat16, window, weight_half=2.0 ** -8)


def test_many_requests(ops):
    """More requests than a warp has lanes, with lengths far apart: ranges that hold parts of several pairs."""
    rng = np.random.default_rng(6)
    lens = [int(x) for x in np.exp(rng.uniform(0, np.log(900), 75))]
    for hd, heads, kv_heads in ((128, 6, 2), (64, 4, 4)):
        cache = Cache(ops, lens, kv_heads, hd, 16, seed=23)
        check_attention(ops, cache, [1] * 75, heads, torch.bfloat16)
        check_attention(ops, cache, [min(l, 1 + i % 5) for i, l in enumerate(lens)], heads, torch.bfloat16, weight_half=2.0 ** -8)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales(ops, scale):
    cache = Cache(ops, [70, 300], 2, 128, 16, seed=24)
    for dtype in DTYPES:
        check_attention(ops, cache, [1, 4], 6, dtype, scale=scale, weight_half=2.0 ** -8)


def test_pages_gigabytes_apart(ops):
    """A pool of more than 2**32 bytes: rows written to, read from and attended over in its first and last pages."""
    kv_heads, hd, heads = 2, 128, 6
    record = q4.parts(16, hd, hd, 2)[1]
    n_pages = 2 ** 32 // (kv_heads * record) + 40
    pool = torch.zeros(n_pages + 1, 1, kv_heads * record, dtype=torch.uint8, device=DEV)
    table = i32([[n_pages - 1, 3, n_pages - 7, 0]])
    for ps, view in ((16, ops.KvView(pool, table, 0, 16, kv_heads, hd, bits=4)),):
        n = 60
        qkv = torch.randn(n, (heads + 2 * kv_heads) * hd, generator=torch.Generator().manual_seed(3)).to(DEV)
        q = torch.empty(n, heads * hd, dtype=torch.bfloat16, device=DEV)
        ops.rope_kv_write(qkv, None, i32(range(n)), i32([0] * n), q, view, heads, 0)
        k = torch.empty(n, kv_heads, hd, device=DEV)
        v = torch.empty_like(k)
        ops.kv_read(view, i32([[0], [0], [n], [0]]), k, v)
        x = qkv.cpu().numpy()[:, heads * hd:].reshape(n, 2 * kv_heads, hd)
        want = q4.values(*q4.quantise(x))
        assert (k.double().cpu().numpy() == want[:, :kv_heads]).all() and (v.double().cpu().numpy() == want[:, kv_heads:]).all()
        cache = Cache.__new__(Cache)
        cache.lens, cache.kv_heads, cache.hd, cache.v_dim, cache.view = [n], kv_heads, hd, hd, view
        cache.k, cache.v = [want[:, :kv_heads]], [want[:, kv_heads:]]
        for q_len in (1, 5, 60):
            check_attention(ops, cache, [q_len], heads, torch.bfloat16, weight_half=2.0 ** -8)
        check_attention(ops, cache, [2], heads, torch.float32)


def test_checked_tables(ops):
    """With a fault record, an entry beyond the pool is recorded and the sink page used in its place, by every kernel."""
    for hd, heads, kv_heads, dtype, q_lens in ((128, 6, 2, torch.bfloat16, [1]), (128, 28, 4, torch.bfloat16, [300]), (48, 3, 3, torch.float32, [1])):
        cache = Cache(ops, [300], kv_heads, hd, 16, seed=25)
        n_pages = cache.pool.shape[0] - 1
        fault = torch.zeros(2, dtype=torch.int32, device=DEV)
        view = ops.KvView(cache.pool, cache.dev_table, 1, 16, kv_heads, hd, bits=4, fault=fault)
        cache.view = view
        attend(ops, cache, q_lens, heads, dtype)
        assert fault.tolist() == [0, 0]
        plain = attend(ops, cache, q_lens, heads, dtype)[0].clone()
        cache.view = ops.KvView(cache.pool, cache.dev_table, 1, 16, kv_heads, hd, bits=4)
        assert torch.equal(attend(ops, cache, q_lens, heads, dtype)[0], plain)
        cache.view = view
        cache.pool[n_pages] = 0                           # the sink: finite
        for bad in (n_pages + 5, -3):
            cache.dev_table[0, 2] = bad
            attend(ops, cache, q_lens, heads, dtype)
            assert fault.tolist() == [1, bad]
            fault.zero_()
            ops.kv_read(view, i32([[0], [32], [4], [0]]), torch.empty(4, kv_heads, hd, device=DEV))
            assert fault.tolist() == [1, bad]
            fault.zero_()
            before = cache.pool[:n_pages].clone()
            for rot in (0, hd):
                tab = torch.from_numpy(rope([33], hd)).to(DEV) if rot else None
                ops.rope_kv_write(torch.ones(1, (heads + 2 * kv_heads) * hd, device=DEV), tab, i32([33]), i32([0]),
                                  torch.empty(1, heads * hd, dtype=dtype, device=DEV), view, heads, rot)
                assert fault.tolist() == [1, bad] and torch.equal(cache.pool[:n_pages], before)
                fault.zero_()


def test_prompts_read_back_in_groups(ops, monkeypatch):
    """More positions than are read back at a time: groups of requests one after another."""
    from axon_b200.kernels import fast
    monkeypatch.setattr(fast, "Q4_PROMPT_POSITIONS", 700)
    cache = Cache(ops, [300, 300, 900, 150, 333], 2, 128, 16, seed=22)
    check_attention(ops, cache, [300, 200, 150, 150, 1], 6, torch.bfloat16, weight_half=2.0 ** -8)


def force(monkeypatch, way):
    """Make every segment of more than 64 query rows go one way."""
    from axon_b200.kernels import fast
    monkeypatch.setattr(fast, "Q4_LONG_START" if way == "read back" else "Q4_SHORT_START", -1e9)


@pytest.mark.parametrize("way", ["read back", "4-bit"])
@pytest.mark.parametrize("heads,kv_heads,hd,ps", [(28, 4, 128, 16), (6, 2, 64, 32), (64, 1, 128, 16), (3, 1, 32, 16), (7, 1, 128, 48)])
@pytest.mark.parametrize("window", [0, 100])
def test_prompts_by_either_way(ops, monkeypatch, way, heads, kv_heads, hd, ps, window):
    force(monkeypatch, way)
    cache = Cache(ops, [300, 700, 41, 1, 650, 129], kv_heads, hd, ps, window=window, seed=26, loud=0.5)
    for q_lens in ([300, 259, 3, 1, 100, 0], [0, 0, 0, 0, 0, 129], [0, 700, 0, 0, 650, 0], [22, 1, 41, 1, 65, 2]):
        check_attention(ops, cache, q_lens, heads, torch.bfloat16, window, weight_half=2.0 ** -8)


def test_groups_of_prompts(ops, monkeypatch):
    """Prompts read back in several groups, beside portions that are not."""
    from axon_b200.kernels import fast
    force(monkeypatch, "read back")
    monkeypatch.setattr(fast, "Q4_PROMPT_POSITIONS", 700)
    cache = Cache(ops, [300, 300, 900, 150, 333], 2, 128, 16, seed=27)
    out, ctx = check_attention(ops, cache, [300, 200, 150, 150, 1], 6, torch.bfloat16, weight_half=2.0 ** -8)
    plans = next(v[1] for k, v in ctx.scratch.items() if k[0] == "q4_work")
    assert len(plans) == 3


def test_what_is_not_finite_stays_with_who_sees_it(ops):
    """A NaN key or value is NaN for the tokens that see it and for no others, in every head's own channels."""
    for hd, heads, kv_heads in ((128, 6, 2), (64, 4, 4)):
        for bad_key in (True, False):
            cache = Cache(ops, [50, 50], kv_heads, hd, 16, seed=14)
            page, i = int(cache.table[0, 40 // 16]), 40 % 16
            place = cache.places[1 if bad_key else 3]
            cache.pool[page, 1, place[0] + i * place[1]] = 0xFF          # kv head 0, first group, position 40 of request 0
            for k in (1, 4):
                out = attend(ops, cache, [k, k], heads, torch.bfloat16)[0].view(2, k, heads, hd)
                group = heads // kv_heads
                assert torch.isfinite(out[1]).all() and torch.isfinite(out[0, :, group:]).all()
                nan = torch.isnan(out[0, :, :group])
                assert nan.all() if bad_key else nan[..., :16].all() and not nan[..., 16:].any()
    # tokens before the bad one, in the same portion
    cache = Cache(ops, [44], 2, 128, 16, seed=14)
    page, i = int(cache.table[0, 40 // 16]), 40 % 16
    for which in (1, 3):
        cache.pool[page, 1, cache.places[which][0] + i * cache.places[which][1]] = 0xFF
        out = attend(ops, cache, [8], 2, torch.bfloat16)[0].view(8, 2, 128)
        assert torch.isfinite(out[:4]).all() and torch.isnan(out[4:, 0, :16]).all() and torch.isfinite(out[:, 1]).all()


def test_large_queries_and_keys(ops):
    """Scores far apart: one key takes all the weight; and queries that overflow half precision."""
    cache = Cache(ops, [90], 1, 128, 16, seed=15, loud=30.0)
    q = (torch.randn(1, 4 * 128, generator=torch.Generator().manual_seed(1)) * torch.tensor([1e-6, 1.0, 300.0, 2e5]).repeat_interleave(128)).to(torch.bfloat16).to(DEV)
    check_attention(ops, cache, [1], 4, torch.bfloat16, q=q)
    check_attention(ops, cache, [1], 4, torch.float32, q=q.float())
    check_attention(ops, cache, [1], 4, torch.bfloat16, q=torch.zeros_like(q))


def test_one_plane_and_wider_values(ops):
    for v_dim, planes in ((None, 1), (96, 2), (16, 2)):
        cache = Cache(ops, [37, 70], 2, 64, 16, v_dim, planes, seed=16)
        if planes == 1:
            cache.v = cache.k
        for dtype in DTYPES:
            check_attention(ops, cache, [1, 3], 6, dtype)


def test_the_same_call_gives_the_same_bits(ops):
    for q_lens, dtype in (([1, 1, 1], torch.bfloat16), ([5, 1, 40], torch.bfloat16), ([1, 1, 1], torch.float32)):
        cache = Cache(ops, [1500, 40, 300], 2, 128, 16, seed=17)
        first = attend(ops, cache, q_lens, 14, dtype)[0].clone()
        for _ in range(3):
            assert torch.equal(attend(ops, cache, q_lens, 14, dtype)[0], first)


def test_on_another_stream_and_in_a_graph(ops):
    """Launches go to the current stream; a captured write and attention replays on new inputs."""
    from axon_b200.parts.base import Runtime
    rt = Runtime(torch.bfloat16, DEV, kv_bits=4)
    heads, kv_heads, hd = 14, 2, 128
    cache = Cache(ops, [700, 33], kv_heads, hd, 16, seed=18)
    qkv = torch.randn(2, (heads + 2 * kv_heads) * hd, device=DEV)
    pos, slot, q = i32([699, 32]), i32([0, 1]), torch.empty(2, heads * hd, dtype=torch.bfloat16, device=DEV)
    from axon_b200.kernels import linear
    from axon_b200.parts.base import StepContext
    ctx = StepContext(rt=rt, n_tokens=2, tokens=None, positions=pos, token_slot=slot, seg_slot=[0, 1], seg_q_start=[0, 1], seg_q_len=[1, 1],
                      seg_kv_len=[700, 33], segments=i32([[0, 1], [0, 1], [1, 1], [700, 33]]), unit_items=i32([[0, 0], [1, 0]]))
    out = torch.empty(2, heads * hd, dtype=torch.bfloat16, device=DEV)

    def run():
        ops.rope_kv_write(qkv, None, pos, slot, q, cache.view, heads, 0)
        linear.attention(q, cache.view, ctx, out, heads, 0.1)

    run()
    eager = out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out.zero_()
        run()
        on_side = out.clone()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, eager)
    # lists that a kernel on the stream has only just written
    fresh = (ctx.segments, ctx.positions, ctx.token_slot, cache.view.block_table)
    kept = [x.clone() for x in fresh]
    for k in range(20):
        for x, y in zip(fresh, kept):
            x.zero_()
            x.add_(y)
        out.zero_()
        run()
        assert torch.equal(out, eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for k in range(3):
        qkv.copy_(torch.randn_like(qkv))
        graph.replay()
        replayed = out.clone()
        run()
        assert torch.equal(replayed, out)


# -- the engine -------------------------------------------------------------

def engine_for(folder, dtype, **kw):
    from axon_b200.engine.build import build_engine
    kw.setdefault("max_slots", 8)
    kw.setdefault("max_tokens", 512)
    return build_engine(folder, dtype=dtype, kv="q4", **kw)


def logits_over_cached(cfg, w, tokens, cached):
    """Float64 logits of a whole sequence whose layers attend over the given keys and values: what the
    engine must answer from the cache it has, whichever side of a rounding border each value fell on."""
    import plain_qwen2 as plain
    H, hd = cfg["num_attention_heads"], cfg["head_dim"]
    x = plain.embed(w["model.embed_tokens.weight"], tokens)
    fresh = []
    for l in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{l}."
        h = plain.rms_norm(x, w[p + "input_layernorm.weight"], cfg["rms_norm_eps"])
        a = p + "self_attn."
        q = plain.linear(h, w[a + "q_proj.weight"], w[a + "q_proj.bias"]).view(len(tokens), H, hd)
        k = plain.linear(h, w[a + "k_proj.weight"], w[a + "k_proj.bias"]).view(len(tokens), -1, hd)
        v = plain.linear(h, w[a + "v_proj.weight"], w[a + "v_proj.bias"]).view(len(tokens), -1, hd)
        pos = list(range(len(tokens)))
        fresh.append((plain.rope_half(k, pos, cfg["rope_theta"]), v))
        o = plain.causal_gqa_attention(plain.rope_half(q, pos, cfg["rope_theta"]), *cached[l])
        x = x + plain.linear(o.reshape(len(tokens), H * hd), w[a + "o_proj.weight"])
        h = plain.rms_norm(x, w[p + "post_attention_layernorm.weight"], cfg["rms_norm_eps"])
        x = x + plain.swiglu_ffn(h, w[p + "mlp.gate_proj.weight"], w[p + "mlp.up_proj.weight"], w[p + "mlp.down_proj.weight"])
    h = plain.rms_norm(x, w["model.norm.weight"], cfg["rms_norm_eps"])
    head = w["model.embed_tokens.weight"] if cfg["tie_word_embeddings"] else w["lm_head.weight"]
    return plain.linear(h, head), fresh


#: of the largest logit: the engine's own tolerances (float rounding; activations of 8 bits between kernels)
ENGINE_TOL = {"float32": 2e-5, "bfloat16": 3e-2}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
@pytest.mark.parametrize("sizes", [[200], [5, 30, 3, 17, 2, 1, 33], [40, 1, 1, 1, 1, 1, 1, 1]])
def test_engine(model_folders, name, dtype, sizes):
    """Prompts whole, in portions and token by token: the logits of every place against float64 over the same
    cache, and the cache against the float64 keys and values it was quantised from."""
    import plain_qwen2 as plain
    from axon_b200.engine.step import StepEntry
    from test_engine_gpu import tokens_for
    cfg, w = plain.read_model(model_folders[name])
    engine = engine_for(model_folders[name], dtype, page_size=16, shuffle_seed=5)
    lens = [1, 37, 100]
    toks = [tokens_for(name, i, n) for i, n in enumerate(lens)]
    slots = [engine.open_request() for _ in lens]
    got = [[] for _ in lens]
    fed, k = [0] * len(lens), 0
    while any(f < n for f, n in zip(fed, lens)):
        entries, who = [], []
        for i, n in enumerate(lens):
            size = min(sizes[(k + i) % len(sizes)], n - fed[i])
            if size > 0:
                entries.append(StepEntry(slots[i], toks[i][fed[i]:fed[i] + size], range(size)))
                who.append((i, size))
                fed[i] += size
        rows = engine.step(entries).double().cpu()
        for i, size in who:
            got[i].append(rows[:size])
            rows = rows[size:]
        k += 1
    for i, n in enumerate(lens):
        cached = [tuple(t.double().cpu() for t in engine.cache.read(slots[i], l)) for l in range(cfg["num_hidden_layers"])]
        want, fresh = logits_over_cached(cfg, w, toks[i], cached)
        scale = float(want.abs().max())
        err = float((torch.cat(got[i]) - want).abs().max())
        assert err <= ENGINE_TOL[dtype] * scale, f"request {i}: {err / scale:.2e} of the largest logit"
        for (k_c, v_c), (k_f, v_f) in zip(cached, fresh):
            for c, f in ((k_c, k_f), (v_c, v_f)):
                groups = f.unflatten(-1, (-1, 16))
                # half a step of the group (at most 9/8 of its largest value over 7.5), and what the model's dtype moves the value by
                room = groups.abs().amax(-1, keepdim=True) * (1.125 / 7.5 / 2) * (1 + 2 * ENGINE_TOL[dtype]) + ENGINE_TOL[dtype] * float(f.abs().max())
                assert ((c.unflatten(-1, (-1, 16)) - groups).abs() <= room + 2.0 ** -18).all()
    engine.check_device()
    engine.cache.manager.check()


def test_serving_with_a_quantised_cache(model_folders):
    """Through the front door: more requests than slots and few pages (preemption), replayed graphs; alone or in a crowd a request's
    greedy tokens come from the same numbers."""
    import axon_b200 as axon
    from test_engine_gpu import tokens_for
    prompts = [tokens_for("C", i, 10 + 23 * i) for i in range(6)]
    opts = axon.BackendOptions().max_ctx(256).kv("q4").dtype("float32").kv_tokens(320).parallel(3)
    net = axon.Backend(axon.load(model_folders["C"]), opts)
    outs = net.generate_batch(prompts, 24)
    alone = axon.Backend(axon.load(model_folders["C"]), axon.BackendOptions().max_ctx(256).kv("q4").dtype("float32").parallel(1))
    for p, o in zip(prompts, outs):
        assert len(o) == 24
        with alone.new_cache() as cache:
            logits = alone.prefill_logits(p, 0, cache)
            assert axon.generate(alone, cache, p, logits, axon.GenOpts.greedy(24)).ids == o
    full = axon.Backend(axon.load(model_folders["C"]), axon.BackendOptions().max_ctx(256).dtype("float32"))
    assert net.engine.cache.bytes_per_token() * 64 == full.engine.cache.bytes_per_token() * 9


def test_command_line(model_folders):
    import os
    import subprocess
    import sys
    from conftest import ROOT
    run = lambda *a: subprocess.run([sys.executable, os.path.join(ROOT, "bin", "axon"), "gen", model_folders["C"], "1 2 3", "-n", "5", *a],  # noqa: E731
                                    capture_output=True, text=True, timeout=300)
    got = run("--kv", "q4")
    assert got.returncode == 0 and len(got.stdout.split()) >= 5, got.stderr
    bad = run("--kv", "q5")
    assert bad.returncode != 0 and "q5" in bad.stderr


def test_graphs_outlive_longer_contexts(model_folders):
    """Portions of one size at the end of ever longer requests move no buffer that a captured step reads (the engine's own
    buffers follow the tokens of a step, and what a portion reads back follows its context)."""
    from axon_b200.engine.step import StepEntry
    from test_engine_gpu import tokens_for
    e = engine_for(model_folders["C"], "bfloat16", max_tokens=4096, max_positions=1000, max_step_tokens=1000)
    a, b = e.open_request(), e.open_request()
    e.step([StepEntry(b, tokens_for("C", 1, 100), [99])])
    e.step([StepEntry(a, tokens_for("C", 0, 9), [8])])
    for t in range(4):
        e.step([StepEntry(a, [t], [0])])
    graphs = dict(e._graphs)
    assert graphs
    for i in range(8):
        e.step([StepEntry(b, tokens_for("C", 2 + i, 100), [99])])
    e.step([StepEntry(a, [7], [0])])
    assert all(e._graphs.get(k) is g for k, g in graphs.items()), "a captured step was thrown away"


def test_reading_what_a_request_holds(model_folders):
    from axon_b200.engine.build import build_engine
    from axon_b200.engine.step import StepEntry
    from test_engine_gpu import tokens_for
    toks = tokens_for("B", 0, 50)
    held = []
    for kv in ("auto", "q4"):
        e = build_engine(model_folders["B"], dtype="float32", kv=kv, max_slots=2, max_tokens=256, max_positions=128, page_size=8, shuffle_seed=2)
        s = e.open_request()
        e.step([StepEntry(s, toks, [])])
        held.append(e.cache.read(s, 1))
        k, v = e.cache.read(s, 1, first=7, count=20)
        assert torch.equal(k, held[-1][0][7:27]) and torch.equal(v, held[-1][1][7:27])
        for first, count in ((0, 51), (-1, 3), (50, 1)):
            with pytest.raises(ValueError, match="holds positions"):
                e.cache.read(s, 1, first=first, count=count)
        with pytest.raises(ValueError, match="not open"):
            e.cache.read(1 - s, 1)
    assert held[0][0].shape == held[1][0].shape and held[1][0].dtype == torch.float32
    # of layer 0 the two engines quantise the same numbers; of layer 1 the keys have moved by what layer 0's rounding did
    assert float((held[0][0] - held[1][0]).abs().max()) < float(held[0][0].abs().max())


# -- large portions ---------------------------------------------------------

def random_pages(ops, positions, kv_heads, hd, seed, ps=16):
    """One request of many positions whose pages hold random codes and steps of 0.125 to 0.47; the view, its keys and its values."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    n_pages, record = -(-positions // ps), q4.parts(ps, hd, hd, 2)[1]
    pool = torch.randint(0, 256, (n_pages + 1, 1, kv_heads * record), dtype=torch.uint8, device=DEV, generator=g)
    heads = pool.view(n_pages + 1, kv_heads, record)
    for at, row in q4.parts(ps, hd, hd, 2)[0][1::2]:
        heads[:, :, at:at + ps * row] = heads[:, :, at:at + ps * row] & 0x0F | 0x60
    table = torch.randperm(n_pages, generator=g, device=DEV).int().view(1, -1)
    view = ops.KvView(pool, table, 0, ps, kv_heads, hd, bits=4)
    k = torch.empty(positions, kv_heads, hd, device=DEV)
    v = torch.empty_like(k)
    ops.kv_read(view, i32([[0], [0], [positions], [0]]), k, v)
    return view, k, v


def check_rows(out, q, k, v, rows, first, heads, scale, weight_half, window=0):
    """Some rows of a portion whose first token is at position ``first``, against float64 on the device, within
    ``check_attention``'s bound and what 4-bit attention's half-precision queries may lose: rows are scaled to the largest element
    in [1, 2), where halves are off by 2^-25 at most below 2^-14 and hold a bfloat16 element's eight bits above 2^-17."""
    hd, kv_heads = k.shape[2], k.shape[1]
    group = heads // kv_heads
    for h in range(kv_heads):
        kd, vd = k[:, h].double(), v[:, h].double()
        for r in rows:
            n = first + r + 1
            lo = max(0, n - window) if window else 0
            kr, vr = kd[lo:n], vd[lo:n]
            qr = q[r].view(heads, hd)[h * group:(h + 1) * group].double()
            s = qr @ kr.T * scale
            w = torch.softmax(s, -1)
            want, mass = w @ vr, w @ vr.abs()
            e_s = ((qr.abs() @ kr.abs().T).amax(-1) * ((hd + 4) * 2.0 ** -23 + 2.0 ** -22) +
                   qr.abs().amax(-1) * 2.0 ** -25 * kr.abs().sum(-1).amax()) * abs(scale)
            tol = (2.0 ** -25 * vr.abs().sum(0) + mass * (weight_half + 2 * e_s[:, None] + 2.0 ** -20 + (n + 8) * 2.0 ** -23) +
                   1.01 * 2.0 ** -8 * want.abs() + 1e-30)
            err = (out[r].view(heads, hd)[h * group:(h + 1) * group].double() - want).abs()
            assert bool((err <= tol).all()), f"token {r}, kv head {h}: {float((err / tol).max()):.2f} of its bound"


@pytest.mark.parametrize("heads,kv_heads,tokens,end", [(32, 8, 4096, 39936), (64, 8, 2048, 38912)])
def test_portions_of_very_many_items(ops, heads, kv_heads, tokens, end):
    """Heads of 256 take 8 query rows an item: 16,384 pairs of items and kv heads, whose ranges once wrapped in 32 bits."""
    from axon_b200.kernels import linear
    from axon_b200.parts.base import Runtime, StepContext
    view, k, v = random_pages(ops, end, kv_heads, 256, 31)
    q = (torch.randn(tokens, heads * 256, generator=torch.Generator().manual_seed(5)) * 0.5).bfloat16().to(DEV)
    out = torch.full_like(q, float("nan"))
    ctx = StepContext(rt=Runtime(torch.bfloat16, DEV, kv_bits=4), n_tokens=tokens, tokens=None, positions=i32(range(end - tokens, end)),
                      token_slot=i32([0] * tokens), seg_slot=[0], seg_q_start=[0], seg_q_len=[tokens], seg_kv_len=[end],
                      segments=i32([[0], [0], [tokens], [end]]))
    linear.attention(q, view, ctx, out, heads, 1 / 16)
    assert bool(torch.isfinite(out).all()), "rows were left as they were"
    rows = [0, tokens - 1] + np.random.default_rng(2).integers(0, tokens, 14).tolist()
    check_rows(out, q, k, v, rows, end - tokens, heads, 1 / 16, 2.0 ** -11)
    # nothing of that division is left for the next launch
    again = torch.full_like(q, float("nan"))
    linear.attention(q, view, ctx, again, heads, 1 / 16)
    assert torch.equal(again, out)


# -- lists that are a kernel's work -----------------------------------------

def picks(values):
    """Logits whose argmax is ``values`` [n], in rows long enough that the kernel that finds them runs for a while after it has let
    its successor start."""
    v = torch.tensor(np.asarray(values).reshape(-1))
    logits = torch.zeros(len(v), 400_000, device=DEV)
    logits[torch.arange(len(v)), v.to(DEV)] = 1.0
    return logits


def test_positions_slots_and_tables_just_written_by_a_kernel(ops):
    """What a launch just before has still to write is waited for: by the write, the attention's both ways and the plain kernels."""
    from axon_b200.kernels import linear
    from axon_b200.parts.base import Runtime, StepContext
    heads, kv_heads, hd = 14, 2, 128
    cache = Cache(ops, [700, 650], kv_heads, hd, 16, seed=33)
    rt = Runtime(torch.bfloat16, DEV, kv_bits=4)
    table_logits = picks(cache.table)
    table = torch.zeros_like(cache.dev_table)
    view = ops.KvView(cache.pool, table, 1, 16, kv_heads, hd, bits=4)

    # the write: positions, slots, table
    tab = torch.from_numpy(rope([690, 33], hd)).to(DEV)
    qkv = torch.randn(2, (heads + 2 * kv_heads) * hd, generator=torch.Generator().manual_seed(2)).to(DEV)
    q = torch.empty(2, heads * hd, dtype=torch.bfloat16, device=DEV)
    for late in ("positions", "slots", "table"):
        pool = cache.pool.clone()
        ops.rope_kv_write(qkv, tab, i32([690, 33]), i32([0, 1]), q, ops.KvView(pool, cache.dev_table, 1, 16, kv_heads, hd, bits=4), heads, hd)
        got = cache.pool.clone()
        x = {"positions": i32([0, 0]), "slots": i32([1, 0]), "table": table.zero_()}
        fine = {"positions": i32([690, 33]), "slots": i32([0, 1]), "table": cache.dev_table}
        logits = {"positions": picks([690, 33]), "slots": picks([0, 1]), "table": table_logits}[late]
        torch.cuda.synchronize()
        ops.argmax(logits, x[late].view(-1))
        use = {**fine, late: x[late]}
        ops.rope_kv_write(qkv, tab, use["positions"], use["slots"], q, ops.KvView(got, use["table"], 1, 16, kv_heads, hd, bits=4), heads, hd)
        assert torch.equal(got, pool), f"{late} were read too early"

    # attention: segments and table, single tokens, portions and prompts read back
    for q_lens in ([1, 1], [4, 3], [300, 650]):
        n = sum(q_lens)
        want, _, qs, pos, slot, scale = attend(ops, cache, q_lens, heads, torch.bfloat16)
        seg = np.array([[0, 1], [0, q_lens[0]], q_lens, cache.lens])
        for late in ("segments", "table"):
            segments = i32([[0, 0], [0, 0], [1, 1], [1, 1]]) if late == "segments" else i32(seg)
            table.zero_() if late == "table" else table.copy_(cache.dev_table)
            logits = picks(seg) if late == "segments" else table_logits
            ctx = StepContext(rt=rt, n_tokens=n, tokens=None, positions=i32(pos), token_slot=i32(slot), seg_slot=[0, 1], seg_q_start=[0, q_lens[0]],
                              seg_q_len=list(q_lens), seg_kv_len=list(cache.lens), segments=segments)
            out = torch.zeros_like(want)
            linear.attention(qs, cache.view, ctx, out, heads, scale)             # (lists and scratch of this shape are there from now on)
            torch.cuda.synchronize()
            out.zero_()
            ops.argmax(logits, (segments if late == "segments" else table).view(-1))
            linear.attention(qs, view, ctx, out, heads, scale)
            assert torch.equal(out, want), f"{late} were read too early by portions of {q_lens}"
    # the plain kernels, and reading back
    cache32 = attend(ops, cache, [1, 1], heads, torch.float32)
    table.zero_()
    torch.cuda.synchronize()
    ops.argmax(table_logits, table.view(-1))
    out = torch.empty_like(cache32[0])
    ops.attention_plain(cache32[2], view, i32(cache32[3]), i32(cache32[4]), out, heads, cache32[5])
    again = torch.empty_like(out)
    ops.attention_plain(cache32[2], cache.view, i32(cache32[3]), i32(cache32[4]), again, heads, cache32[5])
    assert torch.equal(out, again)
    table.zero_()
    torch.cuda.synchronize()
    ops.argmax(table_logits, table.view(-1))
    keys = torch.empty(650, kv_heads, hd, device=DEV)
    ops.kv_read(view, i32([[1], [0], [650], [0]]), keys)
    assert (keys.double().cpu().numpy() == cache.k[1]).all()


def test_a_step_of_the_engine_is_staged(model_folders):
    """The engine copies what a step's kernels read before the first of them, and says so; a context made by hand does not."""
    from axon_b200.engine.step import StepEntry
    from axon_b200.parts.base import StepContext
    assert StepContext.__dataclass_fields__["staged"].default is False
    e = engine_for(model_folders["C"], "bfloat16")
    e.cuda_graphs = False
    seen, forward = [], e.model.forward
    e.model.forward = lambda ctx, *a, **kw: (seen.append(ctx.staged), forward(ctx, *a, **kw))[1]
    e.step([StepEntry(e.open_request(), [1, 2, 3], [2])])
    assert seen == [True]


def test_pieces_are_folded_when_all_have_arrived(ops):
    """Requests cut into many pieces, two sets of queries in turn: scratch holds the other call's pieces whenever a CTA folds, and a
    piece read before it arrived would show in the bits."""
    from axon_b200.kernels import linear
    from axon_b200.parts.base import Runtime, StepContext
    for positions, heads, kv_heads in ((32768, 12, 2), (9001, 28, 4), (700, 14, 2)):
        view, _, _ = random_pages(ops, positions, kv_heads, 128, 41)
        ctx = StepContext(rt=Runtime(torch.bfloat16, DEV, kv_bits=4), n_tokens=1, tokens=None, positions=i32([positions - 1]), token_slot=i32([0]),
                          seg_slot=[0], seg_q_start=[0], seg_q_len=[1], seg_kv_len=[positions], segments=i32([[0], [0], [1], [positions]]))
        qs = [(torch.randn(1, heads * 128, generator=torch.Generator().manual_seed(s)) * 0.3).bfloat16().to(DEV) for s in (1, 2)]
        outs = [torch.zeros_like(q) for q in qs]
        for q, o in zip(qs, outs):
            linear.attention(q, view, ctx, o, heads, 0.09)
        assert torch.isfinite(outs[0]).all() and not torch.equal(*outs)
        got = torch.zeros(300, 2, heads * 128, dtype=torch.bfloat16, device=DEV)
        for k in range(300):
            for j in range(2):
                linear.attention(qs[j], view, ctx, got[k, j:j + 1], heads, 0.09)
        assert all(bool((got[:, j] == outs[j]).all()) for j in range(2))


@pytest.mark.parametrize("name,dtype", [("C", "float32"), ("D", "bfloat16")])
def test_graphs_of_the_plain_kernels_outlive_longer_contexts(model_folders, name, dtype):
    """Decoding beside ever longer contexts moves no buffer of a captured step, and captures few steps."""
    from axon_b200.engine.step import StepEntry
    from test_engine_gpu import tokens_for
    e = engine_for(model_folders[name], dtype, max_tokens=4096, max_positions=2100, max_step_tokens=1000)
    a, b = e.open_request(), e.open_request()
    e.step([StepEntry(a, tokens_for(name, 0, 200), [199])])
    e.step([StepEntry(b, tokens_for(name, 0, 200), [199])])
    captured = []
    for i in range(18):
        e.step([StepEntry(b, tokens_for(name, 2 + i, 100), [99])])
        e.step([StepEntry(a, [1], [0]), StepEntry(b, [2], [0])])
        captured.append(dict(e._graphs))
    for graphs in captured:
        assert all(e._graphs.get(k) is g for k, g in graphs.items()), "a captured step was thrown away"
    assert captured[0] and sum(k[0] == 2 for k in e._graphs) <= 12


def test_prompts_take_no_memory_that_was_not_there(model_folders, monkeypatch):
    """An engine over a 4-bit cache has what its longest prompts are read back into from the start, and the 32-bit model nothing."""
    from axon_b200.engine.step import StepEntry
    from test_engine_gpu import tokens_for
    force(monkeypatch, "read back")
    for dtype in ("bfloat16", "float32"):
        e = engine_for(model_folders["C"], dtype, max_tokens=4096, max_positions=1500, max_step_tokens=3000, max_slots=2)
        held = {k: v.data_ptr() for k, v in e.rt._buffers.items() if k.startswith("q4_prompt_pages")}
        assert len(held) == (dtype == "bfloat16")
        slots = [e.open_request(), e.open_request()]
        e.step([StepEntry(s, tokens_for("C", i, 1500), [1499]) for i, s in enumerate(slots)])
        took = any(k.startswith("q4_plan") for k in e.rt._buffers)
        assert took == (dtype == "bfloat16"), "the prompts should have been read back in the bfloat16 model"
        assert {k: v.data_ptr() for k, v in e.rt._buffers.items() if k.startswith("q4_prompt_pages")} == held


@pytest.mark.parametrize("bits", [0, 4])
@pytest.mark.parametrize("window,n", [(17, 50), (17, 48), (17, 40), (1, 24), (1, 25), (64, 50), (9, 8), (9, 9)])
def test_reading_a_part_with_a_window(ops, bits, window, n):
    """By default what the next token can see; whatever lies in pages that are still held on demand, and nothing given back."""
    from axon_b200.cache.manager import PagedCache
    from axon_b200.parts.spec import KvNeed
    ps, kv_heads, hd = 8, 2, 32
    cache = PagedCache([{"mixer": KvNeed(kv_heads, hd, window=window, bits=bits)}], torch.float32, DEV, page_size=ps, max_tokens=128, max_slots=2,
                       max_positions=64, shuffle_seed=3)
    slot, other = cache.open(), cache.open()
    qkv = torch.randn(n, 3 * kv_heads * hd, generator=torch.Generator().manual_seed(n)).to(DEV)
    kv = qkv.view(n, 3, kv_heads, hd)[:, 1:].cpu().numpy()
    want = q4.values(*q4.quantise(kv)) if bits else kv.astype(np.float64)
    fill = torch.full_like(qkv, 9.0)
    for at in range(n):                       # token by token; another request takes the pages that are given back
        for s, rows in ((slot, qkv), (other, fill)):
            assert cache.reserve(s, at + 1)
            cache.sync_tables()
            ops.rope_kv_write(rows[at:at + 1], None, i32([at]), i32([s]), torch.empty(1, kv_heads * hd, device=DEV), cache.view(0), kv_heads, 0)
            cache.commit(s, at + 1)
            cache.flush()
    seen = max(0, n - window + 1)
    held = seen // ps * ps
    k, v = cache.read(slot, 0)
    assert k.shape[0] == n - seen and k.dtype == torch.float32
    for first in range(held, n + 1):
        k, v = cache.read(slot, 0, first=first)
        assert (k.double().cpu().numpy() == want[first:, 0]).all() and (v.double().cpu().numpy() == want[first:, 1]).all()
    for first in range(-1, held):
        with pytest.raises(ValueError, match="holds positions"):
            cache.read(slot, 0, first=first, count=1)


def test_attention_refuses_operands_that_it_would_read_past(ops):
    from axon_b200.kernels import linear
    from axon_b200.parts.base import Runtime, StepContext
    cache = Cache(ops, [20, 30], 2, 64, 16)
    q, pos, slot = torch.zeros(2, 4 * 64, device=DEV), i32([19, 29]), i32([0, 1])
    out = torch.full_like(q, -7.0)
    for bad in ((pos.long(), slot), (pos, slot.long()), (pos[:1].contiguous(), slot), (pos, slot[:1].contiguous())):
        with pytest.raises(ValueError, match="position and slot"):
            ops.attention_plain(q, cache.view, *bad, out, 4, 0.1)
    scratch, arrived = torch.zeros(4096, device=DEV), torch.zeros(64, dtype=torch.int32, device=DEV)
    for shares in (ops.KeyShares(2, scratch.double(), arrived), ops.KeyShares(2, scratch, arrived.long()), ops.KeyShares(2, scratch), ops.KeyShares(2, None, arrived)):
        with pytest.raises(ValueError, match="scratch and int32 counters"):
            ops.attention_plain(q, cache.view, pos, slot, out, 4, 0.1, shares=shares)
    with pytest.raises(ValueError, match="contiguous CUDA"):
        ops.attention_plain(q, cache.view, pos, slot, out, 4, 0.1, shares=ops.KeyShares(2, scratch.cpu(), arrived))
    assert (out == -7.0).all()
    seg = [[0, 1], [0, 1], [1, 1], [20, 30]]
    good = dict(rt=Runtime(torch.bfloat16, DEV, kv_bits=4), n_tokens=2, tokens=None, positions=pos, token_slot=slot, seg_slot=seg[0], seg_q_start=seg[1],
                seg_q_len=seg[2], seg_kv_len=seg[3], segments=i32(seg))
    qb, ob = q.bfloat16(), torch.full_like(q, -7.0, dtype=torch.bfloat16)
    for change, what in ((dict(segments=i32(seg).long()), "int64"), (dict(segments=i32(seg)[:3].contiguous()), r"\[3, 2\]"),
                         (dict(segments=i32(seg).cpu()), "on cpu"), (dict(segments=i32(seg).T.contiguous().T), "contiguous"),
                         (dict(seg_q_len=[1, 31]), "do not fit"), (dict(seg_q_len=[1, 2]), "do not fit")):
        with pytest.raises(ValueError, match=what):
            linear.attention(qb, cache.view, StepContext(**{**good, **change}), ob, 4, 0.1)
    assert (ob == -7.0).all()
    linear.attention(qb, cache.view, StepContext(**good), ob, 4, 0.1)
    assert torch.isfinite(ob).all() and (ob != -7.0).any()


@pytest.mark.parametrize("way", ["read back", "4-bit"])
@pytest.mark.parametrize("heads,kv_heads,hd", [(14, 2, 128), (6, 2, 64), (6, 2, 32)])
@pytest.mark.parametrize("window", [0, 60])
def test_what_is_not_finite_in_a_prompt_stays_with_who_sees_it(ops, monkeypatch, way, heads, kv_heads, hd, window):
    """A NaN key or value anywhere in a prompt, or before a portion: tokens that do not see it have the bits they have without it,
    whichever way the portion takes; those that see it have NaN in its channels, and no other head has any."""
    if way == "4-bit" and hd == 32:
        return
    force(monkeypatch, way)
    group = heads // kv_heads
    for total, q_len in ((300, 300), (300, 130)):
        for at in (0, 63, 64, 200, 255, 299):
            for part in (1, 3):
                cache = Cache(ops, [total, 70], kv_heads, hd, 16, window=window, seed=35)
                clean = attend(ops, cache, [q_len, 70], heads, torch.bfloat16)[0].clone().view(-1, heads, hd)
                page, i = int(cache.table[0, at // 16]), at % 16
                cache.pool[page, 1, cache.record + cache.places[part][0] + i * cache.places[part][1]] = 0xFF       # kv head 1, its first group
                out = attend(ops, cache, [q_len, 70], heads, torch.bfloat16)[0].view(-1, heads, hd)
                pos = torch.arange(total - q_len, total, device=DEV)
                sees = (pos >= at) & ((pos - at < window) if window else True)
                assert torch.equal(out[q_len:], clean[q_len:]), "another request"
                assert torch.equal(out[:q_len, :group], clean[:q_len, :group]), "another kv head"
                assert torch.equal(out[:q_len][~sees], clean[:q_len][~sees]), f"a token that does not see position {at}"
                assert torch.isnan(out[:q_len][sees][:, group:, :16]).all(), f"a token that sees position {at}"


# -- the 4-bit kernel's own bound -------------------------------------------

def check_tight(ops, cache, q_lens, heads, window=0, **kw):
    """Every token against float64 with weights of eleven bits, which the 4-bit kernel's are and bfloat16's are not."""
    out, _, q, pos, slot, scale = attend(ops, cache, q_lens, heads, torch.bfloat16, window, **kw)
    at = 0
    for s, n in enumerate(q_lens):
        if n:
            k, v = torch.from_numpy(cache.k[s]).to(DEV), torch.from_numpy(cache.v[s]).to(DEV)
            check_rows(out[at:at + n], q[at:at + n], k, v, range(n), cache.lens[s] - n, heads, scale, 2.0 ** -11, window)
        at += n


TIGHT = [l for l in LAYOUTS if l[2] in (64, 128, 256) and l[3] % max(1, 256 // l[2]) == 0]


@pytest.mark.parametrize("heads,kv_heads,hd,ps", TIGHT)
@pytest.mark.parametrize("window", [0, 19])
def test_portions_keep_eleven_bits_of_weights(ops, monkeypatch, heads, kv_heads, hd, ps, window):
    """One, two and four row tiles, with and without a work list; peaked and flat weights."""
    force(monkeypatch, "4-bit")
    cache = Cache(ops, [2, 40, 5, 64, 81, 33], kv_heads, hd, ps, window=window, seed=42)
    for q_lens in ([1, 1, 1, 1, 1, 1], [2, 2, 0, 2, 1, 2], [1, 4, 0, 3, 4, 2], [2, 3, 0, 9, 1, 33]):
        for scale in (None, 1.0):
            check_tight(ops, cache, q_lens, heads, window, scale=scale)


def test_more_portions_keep_eleven_bits_of_weights(ops):
    rng = np.random.default_rng(7)
    lens = [int(x) for x in np.exp(rng.uniform(0, np.log(900), 75))]
    for hd, heads, kv_heads in ((128, 6, 2), (64, 4, 4)):
        check_tight(ops, Cache(ops, lens, kv_heads, hd, 16, seed=43), [min(l, 1 + i % 5) for i, l in enumerate(lens)], heads)
    for scale in (-0.2, 0.0, 3.0):
        check_tight(ops, Cache(ops, [70, 300], 2, 128, 16, seed=44), [1, 4], 6, scale=scale)
    check_tight(ops, Cache(ops, [5003], 4, 128, 16, seed=45, loud=1.0), [4], 28)
    check_tight(ops, Cache(ops, [5003], 4, 128, 16, seed=45, loud=1.0, window=1000), [4], 28, 1000)


def test_queries_that_span_many_powers_of_two(ops):
    """A row's largest element against others down to 2^-30 of it, where halves no longer hold them exactly."""
    heads, hd = 6, 128
    cache = Cache(ops, [90, 33], 2, hd, 16, seed=46)
    g = torch.Generator().manual_seed(8)
    q = torch.randn(3, heads * hd, generator=g) * torch.exp2(-30.0 * torch.rand(3, heads * hd, generator=g))
    q.view(3, heads, hd)[:, :, 5] = 1.9
    for size in (1.0, 2.0 ** -100, 2.0 ** 60):
        check_tight(ops, cache, [2, 1], heads, q=(q * size).bfloat16().to(DEV), scale=0.5 / size)


@pytest.mark.parametrize("heads,kv_heads,hd,ps", [(14, 2, 128, 16), (8, 1, 128, 1), (6, 2, 64, 32), (3, 1, 32, 16), (5, 5, 48, 16)])
@pytest.mark.parametrize("scale", [0.0, -0.2, -0.0])
@pytest.mark.parametrize("window", [0, 60])
def test_prompts_at_scales_that_are_not_positive(ops, monkeypatch, heads, kv_heads, hd, ps, scale, window):
    """Whichever way their length would send them.  Rows read back meet weights of bfloat16, off by 2^-8 at most."""
    force(monkeypatch, "read back")
    cache = Cache(ops, [300, 3, 90], kv_heads, hd, ps, window=window, seed=47)
    check_attention(ops, cache, [300, 1, 40], heads, torch.bfloat16, window, weight_half=2.0 ** -8, scale=scale)


@pytest.mark.parametrize("hd,ps", [(128, 16), (64, 16), (128, 1), (32, 16), (48, 16), (256, 16)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [0, 1])
def test_calls_with_nothing_to_do(ops, hd, ps, dtype, window):
    """No rows, no spans, no tokens; and segments without tokens, or without positions, beside others in one step."""
    from axon_b200.kernels import linear
    from axon_b200.parts.base import Runtime, StepContext
    heads, kv_heads = 6, 2
    cache = Cache(ops, [300, 64, 20, 40], kv_heads, hd, ps, window=window, seed=48)
    before = cache.pool.clone()
    none = i32([])
    ops.rope_kv_write(torch.empty(0, (heads + 2 * kv_heads) * hd, device=DEV), None, none, none, torch.empty(0, heads * hd, dtype=dtype, device=DEV),
                      cache.view, heads, 0)
    keys = torch.full((3, kv_heads, hd), -5.0, device=DEV)
    ops.kv_read(cache.view, torch.empty(4, 0, dtype=torch.int32, device=DEV), keys)
    ops.kv_read(cache.view, i32([[0], [0], [3], [0]]), keys[:0])
    assert (keys == -5.0).all() and torch.equal(cache.pool, before)
    rt = Runtime(dtype, DEV, kv_bits=4)
    empty = dict(rt=rt, n_tokens=0, tokens=None, positions=none, token_slot=none, seg_slot=[], seg_q_start=[], seg_q_len=[], seg_kv_len=[],
                 segments=torch.empty(4, 0, dtype=torch.int32, device=DEV))
    q = torch.empty(0, heads * hd, dtype=dtype, device=DEV)
    linear.attention(q, cache.view, StepContext(**empty), torch.empty_like(q), heads, 0.1, precise=dtype == torch.float32)
    for q_lens in ([300, 0, 0, 1], [1, 0, 0, 3], [200, 0, 0, 40]):
        want, _, qs, pos, slot, scale = attend(ops, cache, q_lens, heads, dtype)
        seg = [[0, 1, 2, 3], [0, q_lens[0], q_lens[0], q_lens[0]], q_lens, [300, 64, 0, 40]]
        ctx = StepContext(rt=rt, n_tokens=len(pos), tokens=None, positions=i32(pos), token_slot=i32(slot), seg_slot=seg[0], seg_q_start=seg[1],
                          seg_q_len=seg[2], seg_kv_len=seg[3], segments=i32(seg))
        out = torch.full_like(want, float("nan"))
        linear.attention(qs, cache.view, ctx, out, heads, scale, precise=dtype == torch.float32)
        assert torch.allclose(out.float(), want.float(), rtol=2.0 ** -6, atol=2.0 ** -6), q_lens


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("way", ["read back", "4-bit"])
@pytest.mark.parametrize("heads,kv_heads,hd,window,pairing", [(4, 2, 16, None, "adjacent"), (8, 1, 128, 7, "half"), (6, 2, 64, 33, "adjacent"),
                                                              (14, 2, 128, 40, "half"), (3, 3, 48, 1, "half")])
def test_attention_part_over_a_quantised_cache(ops, monkeypatch, dtype, way, heads, kv_heads, hd, window, pairing):
    """The mixer with its rotation, write and attention, in cuts, while a window gives pages back to another request: against
    float64 attention over what the cache took."""
    from axon_b200.cache import PagedCache
    from axon_b200.parts import PartSpec, Runtime, part_class
    from dataclasses import replace
    import plain_qwen2 as plain
    from test_parts_gpu import TOL, commit, make_ctx, rand
    force(monkeypatch, way)
    D, T, ps = 72, 150, 4
    rt = Runtime(dtype, DEV, kv_bits=4)
    spec = PartSpec("attention", {"hidden_size": D, "heads": heads, "kv_heads": kv_heads, "head_dim": hd, "qkv_bias": True, "out_bias": False,
                                  "window": window, "scale": None}, {k: k for k in ("q", "k", "v", "o", "q_bias", "k_bias", "v_bias")},
                    {"position": PartSpec("rope", {"head_dim": hd, "theta": 1e4, "pairing": pairing})})
    cls = part_class("mixer", "attention")
    w = {n: rand(*d.shape, seed=200 + i, std=0.3, dtype=torch.float32 if d.kind == "bias" else dtype) for i, (n, d) in enumerate(cls.tensors(spec).items())}
    ref = {k: v.double().cpu() for k, v in w.items()}
    mixer = cls(spec, dict(w), rt, lambda sub: part_class("position", sub.kind)(sub, {}, rt, None))
    cache = PagedCache([replace(cls.cache_need(spec), bits=4)], dtype, DEV, page_size=ps, max_tokens=400, max_slots=2, max_positions=160, shuffle_seed=3)
    rt.kv_page_size = ps
    hs = [rand(T, D, seed=8 + r, dtype=dtype) for r in range(2)]
    for cuts in ([T], [70, 1, 1, 30, 2, 40, 6], [1] * 9 + [141]):
        slots = [cache.open(), cache.open()]
        outs = [torch.zeros(T, D, device=DEV) for _ in slots]
        held = [([], []) for _ in slots]
        at = 0
        for n in cuts:
            cache.flush()
            ctx = make_ctx(rt, cache, [(s, n) for s in slots])
            xs = torch.zeros(2 * n, D, device=DEV)
            mixer.forward(torch.cat([h[at:at + n] for h in hs]).contiguous(), xs, ctx, cache.view(0), True)
            k, v = (torch.empty(2 * n, kv_heads, hd, dtype=dtype, device=DEV) for _ in range(2))
            ops.kv_read(cache.view(0), i32([slots, [at, at], [n, n], [0, n]]), k, v)
            commit(cache, ctx)
            for r in range(2):
                outs[r][at:at + n] = xs[r * n:(r + 1) * n]
                held[r][0].append(k[r * n:(r + 1) * n].double().cpu())
                held[r][1].append(v[r * n:(r + 1) * n].double().cpu())
            at += n
        for r in range(2):
            q = plain.linear(hs[r].double().cpu(), ref["q"], ref["q_bias"]).view(T, heads, hd)
            q = (plain.rope_half if pairing == "half" else plain_rope_adjacent)(q, range(T), 1e4)
            o = plain.causal_gqa_attention(q, torch.cat(held[r][0]), torch.cat(held[r][1]), window=window)
            want = plain.linear(o.reshape(T, heads * hd), ref["o"])
            err = float((outs[r].double().cpu() - want).abs().max() / want.abs().max())
            assert err <= TOL[dtype], f"request {r}, cuts {cuts}: {err:.2e}"
            cache.close(slots[r])


def plain_rope_adjacent(x, positions, theta):
    """Rotation of pairs (2 i, 2 i + 1) in float64."""
    half = x.shape[-1] // 2
    ang = torch.tensor(list(positions), dtype=torch.float64)[:, None] * theta ** (-torch.arange(half, dtype=torch.float64) / half)[None]
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_capture_wants_the_call_to_have_run_once(ops, dtype):
    """Counters that must be zero are not made inside a capture; after one eager call capture, replay and eager calls mix in any order."""
    from axon_b200.kernels import linear
    from axon_b200.parts.base import Runtime, StepContext
    heads, kv_heads, hd = 14, 2, 128
    cache = Cache(ops, [900, 33], kv_heads, hd, 16, seed=49)
    want, _, q, pos, slot, scale = attend(ops, cache, [1, 1], heads, dtype)
    want = want.clone()
    ctx = StepContext(rt=Runtime(dtype, DEV, kv_bits=4), n_tokens=2, tokens=None, positions=i32(pos), token_slot=i32(slot), seg_slot=[0, 1],
                      seg_q_start=[0, 1], seg_q_len=[1, 1], seg_kv_len=[900, 33], segments=i32([[0, 1], [0, 1], [1, 1], [900, 33]]))
    out = torch.zeros_like(want)

    def run():
        ctx.scratch.clear()
        linear.attention(q, cache.view, ctx, out, heads, scale, precise=dtype == torch.float32)

    with pytest.raises(RuntimeError, match="before it is captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            run()
    run()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for call in (run, graph.replay, run, graph.replay, graph.replay):
        out.zero_()
        call()
        assert torch.equal(out, want)
