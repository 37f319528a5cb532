"""The engine's operations on device tensors, each a hand-written CUDA kernel.

Every function launches on the current CUDA stream and returns nothing: outputs
are tensors the caller passes in.  Tensors must live on the GPU; there is no CPU
path.  ``precise=True`` (the 32-bit model) always takes the plain FFMA kernels; the
bfloat16 model takes the tuned sm_100a kernels where the sizes allow and the plain
ones otherwise.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import torch

from . import lib
from .lib import KvLayout, check
from ..parts.spec import KvNeed

F32, BF16 = 0, 1
_DT = {torch.float32: F32, torch.bfloat16: BF16}


def dtype_code(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError(f"dtype {t.dtype} is not one the kernels take (float32, bfloat16)") from None


def _dev(*tensors: Optional[torch.Tensor]) -> None:
    for t in tensors:
        if t is not None and (not t.is_cuda or not t.is_contiguous()):
            raise ValueError("kernels take contiguous CUDA tensors; there is no CPU path")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


_stream = lib.current_stream


@dataclass
class KvView:
    """One schedule entry's keys and values inside its group's page pool.

    ``pool`` is ``[pages + 1][entries][2][kv_heads][page_size][head_dim]`` (the last
    page is the sink) when keys and values are alike, else ``[pages + 1][entries][elements]``
    with an entry's key plane ``[kv_heads][page_size][head_dim]`` followed, when ``planes``
    is 2, by its value plane ``[kv_heads][page_size][v_dim]``.  With one plane the kernels
    read values from the key plane.  ``block_table`` is the group's device table
    ``[slots][stride]`` of int32.  ``fault`` (two uint32 on the device) switches checked
    tables on: see ``kv_layout.h``.

    With ``bits`` 4 rows are quantised: ``pool`` is uint8 ``[pages + 1][entries][bytes]``, an entry
    holding for each kv head the codes and steps of its key rows and those of its value rows
    (``kv_layout.h``).  :func:`rope_kv_write` quantises what it writes, :func:`kv_read` gives
    positions back as rows, and the attention functions read the pages as they are.
    """

    pool: torch.Tensor
    block_table: torch.Tensor
    entry: int
    page_size: int
    kv_heads: int
    head_dim: int
    window: int = 0
    v_dim: int = 0
    planes: int = 2
    fault: Optional[torch.Tensor] = None
    bits: int = 0

    def __post_init__(self) -> None:
        if self.planes not in (1, 2):
            raise ValueError(f"a cache entry has one or two planes, not {self.planes}")
        self.v_dim = self.head_dim if self.planes == 1 or not self.v_dim else self.v_dim
        entries = self.pool.shape[1]
        if self.bits:
            self._init_quantised(entries)
            return
        self.k_plane = self.kv_heads * self.page_size * self.head_dim
        self.v_plane = self.kv_heads * self.page_size * self.v_dim if self.planes == 2 else 0
        per_entry = self.k_plane + self.v_plane
        if self.pool[0].numel() != entries * per_entry:
            raise ValueError(f"a page of {self.pool[0].numel()} elements does not hold {entries} entries of {per_entry}")
        self.n_pages = self.pool.shape[0] - 1
        self.layout = KvLayout(
            block_table=self.block_table.data_ptr(), table_stride=self.block_table.shape[1],
            page_size=self.page_size, kv_heads=self.kv_heads, head_dim=self.head_dim,
            page_stride=entries * per_entry, entry_offset=self.entry * per_entry,
            v_offset=self.k_plane if self.planes == 2 else 0, v_dim=self.v_dim, planes=self.planes,
            n_pages=self.n_pages, bits=0, fault=None if self.fault is None else self.fault.data_ptr())
        self._ref = ctypes.byref(self.layout)

    def _init_quantised(self, entries: int) -> None:
        need = KvNeed(self.kv_heads, self.head_dim, None, self.v_dim, self.planes, self.bits)
        per_entry = need.page_bytes(self.page_size, 1)
        if self.pool.dtype != torch.uint8 or not self.pool.is_contiguous():
            raise ValueError(f"a {self.bits}-bit pool is contiguous bytes (uint8), not {self.pool.dtype}")
        if self.pool[0].numel() != entries * per_entry:
            raise ValueError(f"a page of {self.pool[0].numel()} bytes does not hold {entries} entries of {per_entry}")
        if self.block_table.dtype != torch.int32 or not self.block_table.is_contiguous():
            raise ValueError("a block table is contiguous int32")
        self.n_pages = self.pool.shape[0] - 1
        self.layout = KvLayout(
            block_table=self.block_table.data_ptr(), table_stride=self.block_table.shape[1],
            page_size=self.page_size, kv_heads=self.kv_heads, head_dim=self.head_dim,
            page_stride=entries * per_entry, entry_offset=self.entry * per_entry, v_offset=0, v_dim=self.v_dim,
            planes=self.planes, n_pages=self.n_pages, bits=self.bits,
            fault=None if self.fault is None else self.fault.data_ptr())
        self._ref = ctypes.byref(self.layout)

    def _plane(self, offset: int, dim: int) -> torch.Tensor:
        if self.bits:
            raise ValueError(f"rows of a {self.bits}-bit cache are no view of its pool: read them with kv_read")
        flat = self.pool.view(self.pool.shape[0], -1)
        start = self.layout.entry_offset + offset
        return flat[:, start:start + self.kv_heads * self.page_size * dim].view(-1, self.kv_heads, self.page_size, dim)

    def keys(self) -> torch.Tensor:
        """This entry's key rows as a view ``[pages + 1][kv_heads][page_size][head_dim]``."""
        return self._plane(0, self.head_dim)

    def values(self) -> torch.Tensor:
        """Its value rows ``[pages + 1][kv_heads][page_size][v_dim]`` (the key rows with one plane)."""
        return self._plane(self.layout.v_offset, self.v_dim)


def embed(tokens: torch.Tensor, table: torch.Tensor, x: torch.Tensor, scale: float = 1.0) -> None:
    _dev(tokens, table, x)
    n, dim = x.shape
    check(lib.cuda().axon_embed(_ptr(tokens), _ptr(table), dtype_code(table), _ptr(x), n, dim, scale, _stream()))


def rmsnorm(x: torch.Tensor, gain: torch.Tensor, out: torch.Tensor, eps: float,
            rows: Optional[torch.Tensor] = None, unit_offset: bool = False, pending=None) -> None:
    """out[r] = norm(x[rows[r]] if rows is given else x[r]); x and gain are float32.

    ``pending`` (a ``fast.PendingFold`` whose output is ``x``): the partial sums that a
    split-K product still owes ``x`` are added to the rows read (and written back) first."""
    _dev(x, gain, out, rows)
    if x.dtype != torch.float32 or gain.dtype != torch.float32:
        raise TypeError("rmsnorm reads a float32 residual and a float32 gain")
    n, dim = out.shape
    if pending is not None:
        pending.claim(x, accumulate=True)
        check(lib.cuda().axon_rmsnorm_fold(_ptr(x), _ptr(gain), _ptr(rows), _ptr(out), dtype_code(out), n, dim,
                                           float(eps), int(unit_offset), _ptr(pending.partial), pending.splits,
                                           pending.ntok, _ptr(pending.bias), _stream()))
        return
    check(lib.cuda().axon_rmsnorm(_ptr(x), _ptr(gain), _ptr(rows), _ptr(out), dtype_code(out), n, dim,
                                  float(eps), int(unit_offset), _stream()))


def fold_partials(pending) -> None:
    """Bring the output of a deferred split-K product up to date (for readers that cannot
    fold the partial sums themselves)."""
    out = pending.out
    accumulate = pending.accumulate
    pending.claim(out, accumulate=accumulate)
    check(lib.cuda().axon_fold_partials(_ptr(pending.partial), pending.splits, pending.ntok, _ptr(pending.bias),
                                        _ptr(out), dtype_code(out), out.shape[0], out.shape[1], out.stride(0),
                                        int(accumulate), _stream()))


def gemm_plain(a: torch.Tensor, w: torch.Tensor, out: torch.Tensor, bias: Optional[torch.Tensor] = None,
               accumulate: bool = False) -> None:
    """out = a @ w.T (+ bias), or out += ... when ``accumulate``; FFMA, any sizes."""
    _dev(a, w, out, bias)
    M, K = a.shape
    N = w.shape[0]
    if w.shape[1] != K or out.shape[0] != M or out.shape[1] != N:
        raise ValueError(f"gemm shapes do not fit: a {tuple(a.shape)} w {tuple(w.shape)} out {tuple(out.shape)}")
    if bias is not None and (bias.dtype != torch.float32 or bias.numel() != N):
        raise ValueError("a bias is float32 with one value per output column")
    check(lib.cuda().axon_gemm_plain(_ptr(a), dtype_code(a), _ptr(w), dtype_code(w), _ptr(bias), _ptr(out),
                                     dtype_code(out), M, N, K, K, N, int(accumulate), _stream()))


def swiglu(gate_up: torch.Tensor, act: torch.Tensor) -> None:
    """act[t][j] = silu(gate_up[t][2j]) * gate_up[t][2j+1]; gate_up is float32."""
    _dev(gate_up, act)
    n, ffn = act.shape
    if gate_up.dtype != torch.float32 or gate_up.shape != (n, 2 * ffn):
        raise ValueError("swiglu reads float32 [n][2 * ffn] with gate and up interleaved")
    check(lib.cuda().axon_swiglu(_ptr(gate_up), _ptr(act), dtype_code(act), n, ffn, _stream()))


def rope_table(positions: torch.Tensor, inv_freq: torch.Tensor, table: torch.Tensor, magnitude: float = 1.0) -> None:
    """table[t][i] = (cos, sin)(positions[t] * inv_freq[i]); inv_freq is float64."""
    _dev(positions, inv_freq, table)
    n, half = table.shape[0], table.shape[1]
    if inv_freq.dtype != torch.float64 or inv_freq.numel() != half or table.dtype != torch.float32:
        raise ValueError("rope_table takes float64 frequencies and writes float32 [n][half][2]")
    check(lib.cuda().axon_rope_table(_ptr(positions), _ptr(inv_freq), _ptr(table), n, half, float(magnitude), _stream()))


def rope_kv_write(qkv: torch.Tensor, table: Optional[torch.Tensor], positions: torch.Tensor,
                  token_slot: torch.Tensor, q_out: torch.Tensor, kv: KvView, heads: int, rot: int,
                  adjacent: bool = False, write_kv: bool = True, pending=None, staged: bool = False) -> None:
    """Rotates queries and keys and writes queries to ``q_out``, keys and values to the cache (quantised
    when ``kv`` has 4 bits).  ``pending`` (a ``fast.PendingFold`` whose output is ``qkv``): the product is
    still in partial sums; they are folded here (with the bias) and ``qkv`` itself is not read.  No two rows of a call may
    name one position of one slot (what it then holds is a mixture of both).  ``staged``:
    positions, slots and the block table were there before the kernels in flight were launched
    (``StepContext.staged``), so that they may be read while the kernel before is still running."""
    if kv.bits:
        quantised("rope_kv_write", kv, qkv, table, positions, token_slot, q_out)
    else:
        _dev(qkv, table, positions, token_slot, q_out, kv.pool)
    n = q_out.shape[0]
    width = (heads + kv.kv_heads) * kv.head_dim + (kv.kv_heads * kv.v_dim if kv.planes == 2 else 0)
    if qkv.dtype != torch.float32 or qkv.shape[1] != width:
        raise ValueError("rope_kv_write reads float32 [n][(heads + kv_heads) * head_dim + kv_heads * v_dim]")
    if kv.bits:
        if q_out.shape[1] != heads * kv.head_dim or qkv.shape[0] < n or positions.numel() < n or token_slot.numel() < n:
            raise ValueError("rope_kv_write takes a row of qkv, a position and a slot for each row of q_out")
        if positions.dtype != torch.int32 or token_slot.dtype != torch.int32:
            raise TypeError("positions and slots are int32")
        if table is not None and (table.dtype != torch.float32 or table.numel() < n * rot):
            raise ValueError("rope_kv_write takes a float32 rotation table [n][rot / 2][2]")
        write, more = lib.cuda().axon_rope_kv_write_q4, (int(staged),)
    else:
        if q_out.dtype != kv.pool.dtype:
            raise TypeError("queries and the cache have one dtype")
        write, more = lib.cuda().axon_rope_kv_write, ()          # (waits in any case)
    if pending is not None:
        pending.claim(qkv, accumulate=False)
    check(write(_ptr(qkv), _ptr(table), _ptr(positions), _ptr(token_slot), _ptr(q_out),
                                        _ptr(kv.pool), dtype_code(q_out), kv._ref, n, heads, rot, int(adjacent),
                                        int(write_kv), None if pending is None else _ptr(pending.partial),
                                        0 if pending is None else pending.splits,
                                        0 if pending is None else pending.ntok,
                                        None if pending is None else _ptr(pending.bias), *more, _stream()))


def quantised(what: str, kv: KvView, *tensors: Optional[torch.Tensor]) -> None:
    """Refuse a view without quantised rows, operands on another device than the one launches go to, and
    operands that are not contiguous."""
    if not kv.bits:
        raise ValueError(f"{what} takes a cache with quantised rows")
    here = torch.cuda.current_device()
    if kv.pool.get_device() != here or kv.block_table.get_device() != here:
        raise ValueError(f"{what}: the cache is on {kv.pool.device}, the current device is cuda:{here}")
    for t in tensors:
        if t is not None and (t.get_device() != here or not t.is_contiguous()):
            raise ValueError(f"{what} takes contiguous CUDA tensors on the current device, cuda:{here}; there is no CPU path"
                             f" (got one on {t.device})")


def kv_read(kv: KvView, spans: torch.Tensor, keys: Optional[torch.Tensor], values: Optional[torch.Tensor] = None) -> None:
    """Positions of requests out of a cache with quantised rows.

    ``spans`` is int32 ``[4][n]``: slot, first position, count and first output row of each span.  Row
    ``r`` of ``keys`` (``[rows][kv_heads][head_dim]``) and of ``values`` (``[rows][kv_heads][v_dim]``), float32 or
    bfloat16, receives the position whose span covers ``r`` (the first such span); the numbers are exact in
    both types.  Rows of no span stay as they are, and so do those of positions outside the block table.
    Either output may be None; with one plane values are the keys."""
    quantised("kv_read", kv, spans, keys, values)
    if spans.dtype != torch.int32 or spans.dim() != 2 or spans.shape[0] != 4:
        raise ValueError("kv_read takes int32 spans [4][n]: slot, first position, count, first output row")
    if keys is None and values is None:
        raise ValueError("kv_read takes keys, values or both to write to")
    rows = (keys if keys is not None else values).shape[0]
    if keys is not None and keys.shape != (rows, kv.kv_heads, kv.head_dim):
        raise ValueError(f"kv_read writes keys as [{rows}][{kv.kv_heads}][{kv.head_dim}], not {list(keys.shape)}")
    if values is not None and values.shape != (rows, kv.kv_heads, kv.v_dim):
        raise ValueError(f"kv_read writes values as [{rows}][{kv.kv_heads}][{kv.v_dim}], not {list(values.shape)}")
    if keys is not None and values is not None and keys.dtype != values.dtype:
        raise TypeError("keys and values are read back in one dtype")
    check(lib.cuda().axon_kv_read_q4(_ptr(kv.pool), kv._ref, _ptr(spans), spans.shape[1], kv.block_table.shape[0], _ptr(keys),
                                     _ptr(values), dtype_code(keys if keys is not None else values), rows, _stream()))


@dataclass
class KeyShares:
    """How the plain attention over a 4-bit cache cuts each token's keys: the number of shares, float32 scratch for their
    results (``axon_attention_q4_plain_scratch``), and int32 counters (zero, and left so), one for each token and eight heads
    of a kv head."""

    count: int = 1
    scratch: Optional[torch.Tensor] = None
    arrived: Optional[torch.Tensor] = None


def attention_plain(q: torch.Tensor, kv: KvView, positions: torch.Tensor, token_slot: torch.Tensor,
                    out: torch.Tensor, heads: int, scale: float, shares: Optional[KeyShares] = None) -> None:
    """Attention of each token over its request's positions up to its own, by the plain kernels.  ``shares``
    (4-bit caches only): into how many shares each token's keys are cut, with their scratch."""
    n = q.shape[0]
    if kv.bits:
        x = shares or KeyShares()
        quantised("attention_plain", kv, q, positions, token_slot, out, x.scratch, x.arrived)
        if out.dtype != q.dtype or out.numel() != n * heads * kv.v_dim or q.numel() != n * heads * kv.head_dim:
            raise ValueError("attention_plain takes queries [n][heads * head_dim] and writes [n][heads * v_dim] in their dtype")
        if positions.dtype != torch.int32 or token_slot.dtype != torch.int32 or positions.numel() < n or token_slot.numel() < n:
            raise ValueError("attention_plain takes an int32 position and slot for each row of queries")
        if x.count > 1 and (x.scratch is None or x.scratch.dtype != torch.float32 or x.arrived is None or x.arrived.dtype != torch.int32):
            raise ValueError("key shares come with float32 scratch and int32 counters")
        check(lib.cuda().axon_attention_q4_plain(_ptr(q), _ptr(kv.pool), dtype_code(q), _ptr(positions), _ptr(token_slot), _ptr(out),
                                                 kv._ref, n, heads, float(scale), int(kv.window), x.count, _ptr(x.scratch),
                                                 0 if x.scratch is None else x.scratch.numel(), _ptr(x.arrived),
                                                 0 if x.arrived is None else x.arrived.numel(), _stream()))
        return
    _dev(q, positions, token_slot, out, kv.pool)
    if q.dtype != kv.pool.dtype or out.dtype != q.dtype:
        raise TypeError("queries, cache and output have one dtype")
    check(lib.cuda().axon_attention_plain(_ptr(q), _ptr(kv.pool), dtype_code(q), _ptr(positions), _ptr(token_slot),
                                          _ptr(out), kv._ref, n, heads, float(scale), int(kv.window), _stream()))


def residual_add(x: torch.Tensor, y: torch.Tensor) -> None:
    _dev(x, y)
    if x.dtype != torch.float32 or x.numel() != y.numel():
        raise ValueError("the residual is float32 and as large as what is added")
    check(lib.cuda().axon_residual_add(_ptr(x), _ptr(y), dtype_code(y), x.numel(), _stream()))


def convert(src: torch.Tensor, dst: torch.Tensor) -> None:
    _dev(src, dst)
    if src.numel() != dst.numel():
        raise ValueError("convert needs equally large tensors")
    check(lib.cuda().axon_convert(_ptr(src), dtype_code(src), _ptr(dst), dtype_code(dst), src.numel(), _stream()))


def argmax(logits: torch.Tensor, best: torch.Tensor, rows: Optional[torch.Tensor] = None) -> None:
    """best[r] = the id of the largest logit of row r, or of row ``rows[r]`` when given."""
    _dev(logits, best, rows)
    n, vocab = best.shape[0], logits.shape[1]
    if rows is None:
        check(lib.cuda().axon_argmax(_ptr(logits), _ptr(best), n, vocab, logits.stride(0), _stream()))
    else:
        check(lib.cuda().axon_argmax_rows(_ptr(logits), _ptr(rows), _ptr(best), n, vocab, logits.stride(0), _stream()))


def gather_rows(src: torch.Tensor, rows: Optional[torch.Tensor], dst: torch.Tensor) -> None:
    """dst[r] = src[rows[r]] (float32 rows; ``rows`` None copies them in order)."""
    _dev(src, rows, dst)
    if src.dtype != torch.float32 or dst.dtype != torch.float32 or dst.shape[1] != src.shape[1]:
        raise ValueError("gather_rows copies float32 rows of one width")
    check(lib.cuda().axon_gather_rows(_ptr(src), _ptr(rows), _ptr(dst), dst.shape[0], dst.shape[1], src.stride(0), _stream()))


def repeat_penalty(logits: torch.Tensor, ids: torch.Tensor, penalty: torch.Tensor) -> None:
    _dev(logits, ids, penalty)
    rows, vocab = logits.shape
    check(lib.cuda().axon_repeat_penalty(_ptr(logits), _ptr(ids), _ptr(penalty), rows, vocab, logits.stride(0),
                                         ids.shape[1], _stream()))


def topk_max() -> int:
    return lib.cuda().axon_topk_max()


def topk(logits: torch.Tensor, ks: torch.Tensor, cand_logit: torch.Tensor, cand_id: torch.Tensor,
         rows: Optional[torch.Tensor] = None) -> None:
    _dev(logits, ks, cand_logit, cand_id, rows)
    n, vocab = ks.shape[0], logits.shape[1]
    check(lib.cuda().axon_topk(_ptr(logits), _ptr(rows), _ptr(ks), _ptr(cand_logit), _ptr(cand_id), n, vocab,
                               logits.stride(0), _stream()))


def sample_temperature(logits: torch.Tensor, temperature: torch.Tensor, uniform: torch.Tensor,
                       picked: torch.Tensor, rows: Optional[torch.Tensor] = None) -> None:
    _dev(logits, temperature, uniform, picked, rows)
    n, vocab = picked.shape[0], logits.shape[1]
    if uniform.dtype != torch.float64 or temperature.dtype != torch.float32:
        raise TypeError("temperatures are float32, uniform numbers float64")
    check(lib.cuda().axon_sample_temperature(_ptr(logits), _ptr(rows), _ptr(temperature), _ptr(uniform), _ptr(picked), n,
                                             vocab, logits.stride(0), _stream()))
