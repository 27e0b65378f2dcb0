"""Attention over the paged cache for steps whose requests share long prefixes: the beams of a
prompt, several answers drawn to one document, requests behind one system prompt.

The keys of a shared prefix are worked through once for all rows of the requests that share it, each
request's own keys for its own rows; both leave partial results, which one more kernel joins
(``csrc/shared_prefix.cu`` has the formulas).  ``plan_shared`` says on the host which tile of rows
works through which range of keys; a plan holds for every step of the same requests, since the kernels
take the ends of the requests' own keys from the step's positions.

The reference computes attention request by request (src/layers/attention.py:35-71) and shares
nothing between requests.
"""

from __future__ import annotations

from dataclasses import dataclass, field

import numpy as np
import torch

from . import library
from .attention import check_head_dim, uses_tensor_cores
from .ops import _check, _need, _on_device, _status_word, _stream, _tag

MAX_SPLITS = 256


@dataclass
class SharedPlan:
    """The work lists of a step's requests: ``items`` by kernel, int32 [n, 8] (``shared_prefix::
    Item``; ``shapes``: their most rows and the unit of their ranges), ``seqs`` int32 [requests, 8] (``shared_prefix::Joined``), ``token_seq`` int32 [tokens];
    ``partial_rows`` rows of partial results.  The arrays are numpy's until ``to`` moves them."""
    items: dict
    shapes: dict
    seqs: "np.ndarray | torch.Tensor"
    token_seq: "np.ndarray | torch.Tensor"
    partial_rows: int
    tokens: int
    device: "torch.device | None" = field(default=None)

    def to(self, device: "torch.device | str") -> "SharedPlan":
        move = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(device)
        seqs = move(self.seqs)
        return SharedPlan({name: move(a) for name, a in self.items.items()}, self.shapes, seqs,
                          move(self.token_seq), self.partial_rows, self.tokens, seqs.device)


@dataclass(frozen=True)
class Tile:
    """A tile of a kernel: the kernel's name among the plan's items, query rows, keys that a range is a
    multiple of (one number for all tiles of a kernel), blocks that fill the device."""
    name: str
    rows: int
    unit: int
    blocks: int


def plan_shared(seq_qlen, group_sizes, prefix_lens, group: int, kv_heads: int, prefix_tile,
                own_tile, tail: int = 0) -> SharedPlan:
    """``seq_qlen``: tokens that each request brings; ``group_sizes``: how many requests, in their
    order, share a prefix; ``prefix_lens``: its keys (0: they share nothing); ``group``: query heads a
    kv head.  ``prefix_tile``: rows -> ``Tile`` for a group of that many rows; ``own_tile`` the same
    for one request's own keys.  ``tail``: about how many keys of its own a request has at most (how
    many ranges they are cut into goes by it, not which keys are seen)."""
    qlen = np.asarray(seq_qlen, dtype=np.int64).reshape(-1)
    sizes = np.asarray(group_sizes, dtype=np.int64).reshape(-1)
    prefix = np.asarray(prefix_lens, dtype=np.int64).reshape(-1)
    _need(bool((qlen >= 0).all()), "shared prefix: a request brings no fewer than 0 tokens")
    _need(len(sizes) == len(prefix) and bool((sizes > 0).all()) and int(sizes.sum()) == len(qlen),
          "shared prefix: group sizes are positive and add up to the requests, with a prefix each")
    _need(bool((prefix >= 0).all()) and int(tail) >= 0, "shared prefix: lengths are not negative")
    total = int(qlen.sum())
    _need(total * group < 1 << 28 and int(prefix.max(initial=0)) < 1 << 31,
          "shared prefix: the step has too many rows or keys")
    tok0 = np.cumsum(qlen) - qlen
    first = np.cumsum(sizes) - sizes
    group_tokens = np.add.reduceat(qlen, first) if len(sizes) else np.zeros(0, dtype=np.int64)
    group_tok0 = tok0[first] if len(sizes) else np.zeros(0, dtype=np.int64)
    # a prefix that only one request's rows read is no different from its own keys
    members = np.add.reduceat((qlen > 0).astype(np.int64), first) if len(sizes) else sizes
    prefix = np.where(members > 1, prefix, 0)
    seqs = np.zeros((len(qlen), 8), dtype=np.int64)
    seqs[:, 0], seqs[:, 1] = tok0, np.repeat(group_tok0, sizes)
    items: dict[str, list] = {}
    shapes: dict[str, tuple] = {}
    base = 0

    def add(t: Tile, part: np.ndarray) -> None:
        items.setdefault(t.name, []).append(part)
        shapes[t.name] = (max(t.rows, shapes.get(t.name, (0, 0))[0]), t.unit)

    # shared keys: ranges of one length for all groups, so long that the blocks fill the device once
    tiles = [prefix_tile(int(t) * group) for t in group_tokens]
    work: dict[str, int] = {}
    for t, p, n in zip(tiles, prefix, group_tokens):
        work[t.name] = work.get(t.name, 0) + -(-int(n) * group // t.rows) * int(p) * kv_heads
    for g, (t, p, n) in enumerate(zip(tiles, prefix, group_tokens)):
        rows, p = int(n) * group, int(p)
        if p == 0 or rows == 0:
            continue
        each = -(-max(work[t.name] // t.blocks, t.unit) // t.unit) * t.unit
        chunks = -(-p // each)
        each = -(-(-(-p // chunks)) // t.unit) * t.unit
        chunks = -(-p // each)
        count = -(-rows // t.rows)
        tile, chunk = np.divmod(np.arange(count * chunks), chunks)
        part = np.zeros((count * chunks, 8), dtype=np.int64)
        part[:, 0], part[:, 2] = group_tok0[g], tile * t.rows
        part[:, 1] = np.minimum(t.rows, rows - part[:, 2])
        part[:, 3], part[:, 4] = first[g], chunk * each
        part[:, 5] = np.minimum(p, (chunk + 1) * each)
        part[:, 7] = base + (tile * chunks + chunk) * t.rows
        # a range after the other, its tiles side by side: they read the same keys
        add(t, part[np.argsort(chunk, kind="stable")])
        members_of = slice(int(first[g]), int(first[g] + sizes[g]))
        seqs[members_of, 2], seqs[members_of, 3], seqs[members_of, 4] = base, chunks, t.rows
        base += count * chunks * t.rows

    # each request's own keys
    live = np.nonzero(qlen > 0)[0]
    if len(live):
        by_tile: dict[Tile, list] = {}
        for s in live:
            by_tile.setdefault(own_tile(int(qlen[s]) * group), []).append(int(s))
        for t, members_of in by_tile.items():
            s = np.asarray(members_of)
            rows = qlen[s] * group
            count = -(-rows // t.rows)
            own = np.maximum(int(tail), qlen[s]) + np.where(np.repeat(prefix, sizes)[s] > 0, 0,
                                                            np.repeat(np.asarray(
                                                                prefix_lens, dtype=np.int64), sizes)[s])
            need = int((count * own).sum()) * kv_heads
            each = max(-(-need // t.blocks), t.unit)
            splits = np.clip(-(-own // each), 1, MAX_SPLITS)
            n = count * splits
            owner = np.repeat(np.arange(len(s)), n)
            at = np.arange(int(n.sum())) - np.repeat(np.cumsum(n) - n, n)
            tile, split = at // splits[owner], at % splits[owner]
            start = base + np.cumsum(n * t.rows) - n * t.rows
            part = np.zeros((len(owner), 8), dtype=np.int64)
            part[:, 0], part[:, 2] = tok0[s[owner]], tile * t.rows
            part[:, 1] = np.minimum(t.rows, rows[owner] - part[:, 2])
            part[:, 3], part[:, 4], part[:, 5] = s[owner], np.repeat(prefix, sizes)[s[owner]], -1
            part[:, 6] = split | splits[owner] << 16
            part[:, 7] = start[owner] + (tile * splits[owner] + split) * t.rows
            add(t, part)
            seqs[s, 5], seqs[s, 6], seqs[s, 7] = start, splits, t.rows
            base += int((n * t.rows).sum())
    _need(base < 1 << 31, "shared prefix: too many partial results")
    return SharedPlan({name: np.concatenate(parts) for name, parts in items.items()}, shapes, seqs,
                      np.repeat(np.arange(len(qlen)), qlen), base, total)


class SharedPrefixAttention:
    """Attention of all layers that share one shape of heads, for steps whose requests share
    prefixes."""

    def __init__(self, dtype: torch.dtype, heads: int, kv_heads: int, head_dim: int, scale: float,
                 device: "torch.device | str | None" = None) -> None:
        """``scale`` above 0; float32 or bfloat16, even head sizes up to 256."""
        check_head_dim(head_dim)
        _tag(dtype)
        if heads <= 0 or kv_heads <= 0 or heads % kv_heads != 0:
            raise ValueError(f"heads ({heads}) must be a multiple of kv_heads ({kv_heads})")
        if not 0.0 < scale < float("inf"):
            raise ValueError(f"shared prefix: the scale must be positive, got {scale}")
        self.dtype, self.heads, self.kv_heads, self.head_dim = dtype, heads, kv_heads, head_dim
        self.scale, self.group = float(scale), heads // kv_heads
        self.tensor_cores = uses_tensor_cores(dtype, head_dim)
        self.mma_module = ("shared_prefix_mma", (f"HEAD_DIM={head_dim}",))
        self._device = None if device is None else torch.device(device)
        self._sms: "int | None" = None

    # ------------------------------------------------------------------ host side
    def _sm_count(self) -> int:
        if self._sms is None:
            device = self._device if self._device is not None else torch.cuda.current_device()
            self._sms = int(torch.cuda.get_device_properties(device).multi_processor_count)
        return self._sms

    def tiles(self) -> "tuple":
        """(rows of a group -> ``Tile``, rows of a request -> ``Tile``)."""
        sms = self._sm_count()
        if self.tensor_cores:
            lib = library.load(*self.mma_module)
            most, blocks = lib.de_shared_mma_rows(), lib.de_shared_mma_blocks_per_sm() * sms
            tile = lambda rows: Tile("mma", min(most, max(1, -(-rows // 16)) * 16), 64, blocks)
            return tile, tile
        plain = Tile("rows", 8, 32, 4 * sms)
        return (lambda rows: plain), (lambda rows: plain)

    def host_plan(self, seq_qlen, group_sizes, prefix_lens, tail: int = 0) -> SharedPlan:
        prefix_tile, own_tile = self.tiles()
        return plan_shared(seq_qlen, group_sizes, prefix_lens, self.group, self.kv_heads, prefix_tile,
                           own_tile, tail)

    def plan(self, seq_qlen, group_sizes, prefix_lens, tail: int = 0) -> SharedPlan:
        """The plan of a step (arguments as ``plan_shared``) on the device.  It holds for every step
        of these requests in which they bring the same numbers of tokens."""
        return self.host_plan(seq_qlen, group_sizes, prefix_lens, tail).to(
            self._device if self._device is not None else "cuda")

    # ------------------------------------------------------------------ device side
    def run(self, q: torch.Tensor, out: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
            block_table: torch.Tensor, seq_slot: torch.Tensor, seq_pos0: torch.Tensor,
            plan: SharedPlan, status: "torch.Tensor | None" = None, buffer=None) -> None:
        """q: a row a token, [heads * d] query features at its front (row stride free), requests in
        the plan's order; out [tokens, heads * d] (row stride free); keys and values [pages,
        kv_heads, page, d], this step's tokens' among them; ``block_table`` [slots, max pages] int32.
        ``seq_slot`` int32: each request's row of the table; the first of a group has the pages of
        the prefix, all have those of their own keys.  ``seq_pos0`` int32: position of each request's
        first token, not before the prefix's end.  A token sees the keys up to its own position; a
        key without a page is not seen and sets ``status`` to 2.  ``buffer(name, shape, dtype)``:
        where the partial results lie during the call (None: fresh memory)."""
        d, tokens = self.head_dim, plan.tokens
        _need(q.dtype == out.dtype == k_pages.dtype == v_pages.dtype == self.dtype,
              "shared prefix: q, out and the pages have the layer's dtype")
        _need(q.dim() == 2 and out.dim() == 2 and q.stride(1) == 1 and out.stride(1) == 1
              and q.shape[0] == out.shape[0] == tokens and q.shape[1] >= self.heads * d
              and out.shape[1] == self.heads * d
              and (tokens < 2 or (q.stride(0) >= self.heads * d and out.stride(0) >= self.heads * d)),
              "shared prefix: q and out have a row a token of the plan, heads * d features each")
        _need(k_pages.dim() == 4 and k_pages.is_contiguous() and v_pages.is_contiguous()
              and k_pages.shape == v_pages.shape and k_pages.shape[1] == self.kv_heads
              and k_pages.shape[3] == d and k_pages.shape[2] > 0,
              "shared prefix: pages must be [pages, kv_heads, page, head_dim]")
        for name, t in (("block_table", block_table), ("seq_slot", seq_slot), ("seq_pos0", seq_pos0)):
            _need(t.dtype == torch.int32 and t.is_contiguous(),
                  f"shared prefix: {name} must be a contiguous int32 tensor")
        _need(block_table.dim() == 2 and seq_slot.shape == seq_pos0.shape == (plan.seqs.shape[0],),
              "shared prefix: block_table [slots, pages], a slot and a position a request")
        _need(plan.device is not None, "shared prefix: the plan is not on the device yet (plan.to)")
        _on_device(q, out, k_pages, v_pages, block_table, seq_slot, seq_pos0, plan.seqs)
        if tokens == 0:
            return
        status = _status_word(status, q)
        make = buffer or (lambda name, shape, dtype: torch.empty(shape, dtype=dtype, device=q.device))
        rows = plan.partial_rows * self.kv_heads
        acc = make("shared_prefix.partial_acc", (rows * d,), torch.float32)
        ml = make("shared_prefix.partial_ml", (rows * 2,), torch.float32)
        lib = library.load("shared_prefix")
        tag = _tag(q.dtype)
        # (rows that are not in 4-byte pieces, pages that are not in 16-byte ones: one by one)
        aligned = not (q.stride(0) % 2 or q.data_ptr() % 4 or k_pages.data_ptr() % 16
                       or v_pages.data_ptr() % 16)
        for name, items in plan.items.items():
            rows, unit = plan.shapes[name]
            before = (q.data_ptr(), q.stride(0), k_pages.data_ptr(), v_pages.data_ptr(),
                      block_table.data_ptr(), block_table.stride(0), k_pages.shape[0],
                      seq_slot.data_ptr(), seq_pos0.data_ptr(), items.data_ptr(), items.shape[0])
            behind = (acc.data_ptr(), ml.data_ptr(), self.heads, self.kv_heads, d, k_pages.shape[2],
                      self.scale, status.data_ptr(), _stream())
            if name == "mma" and aligned:
                _check(library.load(*self.mma_module).de_shared_mma(*before, *behind),
                       "shared prefix attention (mma)")
            else:
                _check(lib.de_shared_rows(tag, *before, rows, unit, *behind),
                       "shared prefix attention")
        _check(lib.de_shared_merge(tag, out.data_ptr(), out.stride(0), plan.token_seq.data_ptr(),
                                   plan.seqs.data_ptr(), acc.data_ptr(), ml.data_ptr(), tokens,
                                   self.heads, self.kv_heads, d, _stream()), "shared prefix merge")
