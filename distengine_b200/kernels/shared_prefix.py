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

from dataclasses import dataclass, field, replace

import numpy as np
import torch

from . import library
from .attention import check_head_dim, uses_tensor_cores
from .ops import _check, _need, _on_device, _status_word, _stream, _tag

MAX_SPLITS = 256         # ranges that a prefix or a request's own keys are cut into


def takes_scale(scale: float) -> bool:
    """Whether the kernels take this scale: above 0, and within the range of float32's normal numbers also
    times log2(e)."""
    return 2.0 ** -126 <= scale <= 2.0 ** 127


@dataclass
class SharedPlan:
    """The work lists of a step's requests: ``items`` by kernel, int32 [n, 8] (``shared_prefix::Item``;
    ``shapes``: their most rows and the unit of their ranges), ``seqs`` int32 [requests, 8]
    (``shared_prefix::Joined``), ``token_seq`` int32 [tokens]; ``partial_rows`` rows of partial results, at
    most ``most_parts`` of one row; ``turns``: some items leave two.  ``group`` query heads a kv head and
    ``kv_heads`` are what the items' rows count: a plan is for layers with these.  The arrays are numpy's
    until ``to`` moves them.  (Kernels read them before the kernel in front of theirs has ended: on the
    device they come from copies, as ``to`` and a step's upload make them.)"""
    items: dict
    shapes: dict
    seqs: "np.ndarray | torch.Tensor"
    token_seq: "np.ndarray | torch.Tensor"
    partial_rows: int
    most_parts: int
    tokens: int
    device: "torch.device | None" = field(default=None)
    turns: bool = False
    group: int = 0
    kv_heads: int = 0

    def to(self, device: "torch.device | str") -> "SharedPlan":
        move = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(device)
        seqs = move(self.seqs)
        return SharedPlan({name: move(a) for name, a in self.items.items()}, self.shapes, seqs,
                          move(self.token_seq), self.partial_rows, self.most_parts, self.tokens, seqs.device,
                          self.turns, self.group, self.kv_heads)


@dataclass(frozen=True)
class Tile:
    """A tile of a kernel: the kernel's name among the plan's items, query rows, keys that a range is a
    multiple of (one number for all tiles of a kernel), blocks (or warps, where those have an item
    each) that the device holds at once; ``places``: partial results that a range leaves; ``least``: keys
    of the shortest range that is worth a block; ``overhead``: keys that take as long as a block's beginning
    and end (tcgen05: 108 rows behind 15,566 keys of 32 kv heads 86 us with 512, 92 with 256); ``own_key``:
    a block has an SM to itself, and this is what a request's own key for 16 rows takes of an SM in keys of
    this tile (64 requests behind 8,192 keys with 500 of their own 45 us with 64 blocks and the own keys'
    beside them, 50 with 128 and those behind them; 43 + 43 behind 463 with 242 21 and 28)."""
    name: str
    rows: int
    unit: int
    blocks: int
    places: int = 1
    least: int = 1
    overhead: int = 256
    own_key: float = 0.0


def choose_range(lengths: np.ndarray, copies: np.ndarray, tile: Tile,
                 beside: float = 0.0) -> "tuple[int, float]":
    """How long the ranges are that ``lengths`` are cut into, a multiple of the tile's unit, and how much of
    the device they leave to others meanwhile: each range of length i is the work of ``copies[i]`` blocks.
    Of all numbers of rounds of as many blocks as the device holds the one that is done first, a block
    costing its keys and the tile's ``overhead``.  ``beside``: work of another kernel, in keys, whose blocks
    find no room beside these: either it follows, or there are so few of these that both are done at
    about the same time."""
    longest, unit, blocks = int(lengths.max(initial=0)), tile.unit, tile.blocks
    whole = -(-longest // unit) * unit
    fewest = max(1, -(-longest // (MAX_SPLITS * unit)), -(-min(tile.least, whole) // unit))
    count = lambda each: int((-(-lengths // each) * copies).sum())

    def shortest(most: int) -> int:                       # of which there are no more
        low, high = fewest, max(whole // unit, fewest)
        while low < high:
            mid = (low + high) // 2
            if count(mid * unit) <= most:
                high = mid
            else:
                low = mid + 1
        return low * unit

    best = None
    least = max(-(-count(max(whole, unit)) // blocks), 1)
    for rounds in range(least, least + 4):
        each = shortest(rounds * blocks)
        cost = rounds * (each + tile.overhead) + beside / blocks
        if best is None or cost < best[0]:
            best = (cost, each, 0.0)
    if beside > 0:
        for eighths in range(6, 0, -1):
            each = shortest(blocks * eighths // 8)
            n = count(each)
            cost = max(each + tile.overhead, beside / max(blocks - n, 1))
            if n <= blocks * 3 // 4 and cost < best[0]:
                best = (cost, each, 1 - n / blocks)
    return best[1:]


def plan_shared(seq_qlen, group_sizes, prefix_lens, group: int, kv_heads: int, prefix_tile,
                own_tile, tail: int = 0) -> SharedPlan:
    """``seq_qlen``: tokens that each request brings; ``group_sizes``: how many requests, in their
    order, share a prefix; ``prefix_lens``: its keys (0: they share nothing); ``group``: query heads a
    kv head.  ``prefix_tile``: (rows, keys) -> ``Tile`` for a group of that many rows and its prefix;
    ``own_tile`` the same for one request's own keys.  ``tail``: about how many keys of
    its own a request has at most (how many ranges they are cut into goes by it, not which keys are
    seen)."""
    qlen = np.asarray(seq_qlen, dtype=np.int64).reshape(-1)
    sizes = np.asarray(group_sizes, dtype=np.int64).reshape(-1)
    shared = np.asarray(prefix_lens, dtype=np.int64).reshape(-1)
    _need(bool((qlen >= 0).all()), "shared prefix: a request brings no fewer than 0 tokens")
    _need(len(sizes) == len(shared) and bool((sizes > 0).all()) and int(sizes.sum()) == len(qlen),
          "shared prefix: group sizes are positive and add up to the requests, with a prefix each")
    _need(bool((shared >= 0).all()) and int(tail) >= 0, "shared prefix: lengths are not negative")
    total = int(qlen.sum())
    _need(total * group < 1 << 28 and int(shared.max(initial=0)) < 1 << 31,
          "shared prefix: the step has too many rows or keys")
    tok0 = np.cumsum(qlen) - qlen
    first = np.cumsum(sizes) - sizes
    live = np.add.reduceat((qlen > 0).astype(np.int64), first) if len(sizes) else sizes
    # a prefix that only one request's rows read is no different from its own keys
    prefix = np.where(live > 1, shared, 0)
    rows = (np.add.reduceat(qlen, first) if len(sizes) else sizes) * group
    seqs = np.zeros((len(qlen), 8), dtype=np.int64)
    seqs[:, 0], seqs[:, 1] = tok0, np.repeat(tok0[first], sizes)
    items: dict[str, list] = {}
    shapes: dict[str, tuple] = {}
    base = 0

    def add(t: Tile, part: np.ndarray) -> None:
        items.setdefault(t.name, []).append(part)
        shapes[t.name] = (max(t.rows, shapes.get(t.name, (0, 0))[0]), t.unit)

    # each request's own keys, behind its prefix
    start = np.repeat(prefix, sizes)
    own = np.maximum(int(tail), qlen) + np.where(start > 0, 0, np.repeat(shared, sizes))
    own_keys = kv_heads * float((own * -(-qlen * group // 16)).sum())

    # shared keys
    by_name: dict[str, list] = {}
    left = 0.0                                            # of the device, beside blocks that have SMs to themselves
    for g in np.nonzero((prefix > 0) & (rows > 0))[0]:
        t = prefix_tile(int(rows[g]), int(prefix[g]))
        by_name.setdefault(t.name, []).append((int(g), t))
    for members in by_name.values():
        lengths = prefix[[g for g, _ in members]]
        copies = np.asarray([-(-int(rows[g]) // t.rows) * kv_heads for g, t in members])
        each, beside = choose_range(lengths, copies, members[0][1], members[0][1].own_key * own_keys)
        left = max(left, beside)
        for g, t in members:
            p, n = int(prefix[g]), int(rows[g])
            chunks, count = -(-p // each), -(-n // t.rows)
            size = -(-(-(-p // chunks)) // t.unit) * t.unit          # ranges of about one length
            chunks = -(-p // size)
            tile, chunk = np.divmod(np.arange(count * chunks), chunks)
            part = np.zeros((count * chunks, 8), dtype=np.int64)
            part[:, 0], part[:, 2] = tok0[first[g]], tile * t.rows
            part[:, 1] = np.minimum(t.rows, n - part[:, 2])
            part[:, 3], part[:, 4] = first[g], chunk * size
            part[:, 5] = np.minimum(p, (chunk + 1) * size)
            part[:, 6] = t.places - 1
            part[:, 7] = base + (tile * chunks + chunk) * t.rows * t.places
            # a range after the other, its tiles side by side: they read the same keys
            add(t, part[np.argsort(chunk, kind="stable")])
            s = slice(int(first[g]), int(first[g] + sizes[g]))
            seqs[s, 2], seqs[s, 3], seqs[s, 4] = base, chunks * t.places, t.rows
            base += count * chunks * t.rows * t.places

    # own keys
    by_tile: dict[Tile, list] = {}
    for s in np.nonzero(qlen > 0)[0]:
        by_tile.setdefault(own_tile(int(qlen[s]) * group, int(own[s])), []).append(int(s))
    for t, members in by_tile.items():
        s = np.asarray(members)
        n = qlen[s] * group
        count = -(-n // t.rows)
        if left:
            t = replace(t, blocks=int(t.blocks * left))
        each, _ = choose_range(own[s], count * kv_heads, t)
        splits = np.clip(-(-own[s] // each), 1, MAX_SPLITS)
        pieces = count * splits
        owner = np.repeat(np.arange(len(s)), pieces)
        at = np.arange(len(owner)) - np.repeat(np.cumsum(pieces) - pieces, pieces)
        tile, split = at // splits[owner], at % splits[owner]
        begin = base + np.cumsum(pieces * t.rows) - pieces * t.rows
        part = np.zeros((len(owner), 8), dtype=np.int64)
        part[:, 0], part[:, 2] = tok0[s[owner]], tile * t.rows
        part[:, 1] = np.minimum(t.rows, n[owner] - part[:, 2])
        part[:, 3], part[:, 4], part[:, 5] = s[owner], start[s[owner]], -1
        part[:, 6] = split | splits[owner] << 16
        part[:, 7] = begin[owner] + (tile * splits[owner] + split) * t.rows
        add(t, part)
        seqs[s, 5], seqs[s, 6], seqs[s, 7] = begin, splits, t.rows
        base += int((pieces * t.rows).sum())
    _need(base < 1 << 31, "shared prefix: too many partial results")
    # (the tcgen05 kernel's blocks first: the others' fill the SMs that those leave)
    names = sorted(items, key=lambda name: (name != "tcgen05", name))
    return SharedPlan({name: np.concatenate(items[name]) for name in names}, shapes, seqs,
                      np.repeat(np.arange(len(qlen)), qlen), base,
                      int((seqs[:, 3] + seqs[:, 6]).max(initial=0)), total,
                      turns=any(t.places > 1 for members in by_name.values() for _, t in members),
                      group=group, kv_heads=kv_heads)


class SharedPrefixAttention:
    """Attention of all layers that share one shape of heads, for steps whose requests share
    prefixes."""

    def __init__(self, dtype: torch.dtype, heads: int, kv_heads: int, head_dim: int, scale: float,
                 device: "torch.device | str | None" = None) -> None:
        """``scale`` above 0 (``takes_scale``); float32 or bfloat16, even head sizes up to 256."""
        check_head_dim(head_dim)
        _tag(dtype)
        if heads <= 0 or kv_heads <= 0 or heads % kv_heads != 0:
            raise ValueError(f"heads ({heads}) must be a multiple of kv_heads ({kv_heads})")
        if not takes_scale(scale):
            raise ValueError(f"shared prefix: the scale must be a positive float32 number, got {scale}")
        self.dtype, self.heads, self.kv_heads, self.head_dim = dtype, heads, kv_heads, head_dim
        self.scale, self.group = float(scale), heads // kv_heads
        self.tensor_cores = uses_tensor_cores(dtype, head_dim)
        self.mma_module = ("shared_prefix_mma", (f"HEAD_DIM={head_dim}",))
        self.tcgen05_module = (("shared_prefix_tcgen05", (f"HEAD_DIM={head_dim}",))
                               if self.tensor_cores and head_dim in (64, 128) else None)
        self._device = None if device is None else torch.device(device)
        self._sms: "int | None" = None

    # ------------------------------------------------------------------ host side
    def _sm_count(self) -> int:
        if self._sms is None:
            device = self._device if self._device is not None else torch.cuda.current_device()
            self._sms = int(torch.cuda.get_device_properties(device).multi_processor_count)
        return self._sms

    def tiles(self, page: "int | None" = None) -> "tuple":
        """(rows of a group, keys that they share) -> ``Tile``, and the same for one request."""
        sms = self._sm_count()
        if self.dtype == torch.float32 and self.head_dim % 4 == 0:
            lib = library.load("shared_prefix_f32")
            tiles = {rows: Tile(f"f32x{rows}", rows, lib.de_shared_f32_unit(),
                                lib.de_shared_f32_held(rows, self.head_dim) * sms)
                     for rows in (8, 16, 32)}
            tile = lambda rows, keys: tiles[8 if rows <= 8 else 16 if rows <= 16 else 32]
            return tile, tile
        if not self.tensor_cores:
            plain = Tile("rows", 8, 32, 4 * sms)
            return (lambda rows, keys: plain), (lambda rows, keys: plain)
        lib = library.load(*self.mma_module)
        unit = lib.de_shared_mma_unit()
        few = Tile("warp", lib.de_shared_mma_rows(), unit, lib.de_shared_mma_held() * sms, least=4 * unit)
        wide = self.tcgen05_module is not None and (
            page is None or library.load(*self.tcgen05_module).de_shared_tcgen05_page_ok(page))

        def shared(rows: int, keys: int) -> Tile:
            # (us, tcgen05 and two tiles of the other: 24 rows, 6 groups behind 1,216 keys of 32 kv heads
            # 55.5 and 39.7; 20 rows behind 2,040 of 8 17.9 and 18.7; 37 rows behind 6,373 of 32 40.6 and,
            # three tiles, 44.2; 48 rows behind 1,214 of 4, head size 64, 16.0 and 12.5)
            if rows > 32 and wide:
                costs = {"overhead": 512, "own_key": self.head_dim / 256}
                return (Tile("tcgen05", 128, 128, sms, 2, least=256, **costs) if rows <= 128 else
                        Tile("tcgen05", 256, 128, sms, **costs))
            return few

        return shared, lambda rows, keys: few

    def host_plan(self, seq_qlen, group_sizes, prefix_lens, tail: int = 0,
                  page: "int | None" = None) -> SharedPlan:
        prefix_tile, own_tile = self.tiles(page)
        return plan_shared(seq_qlen, group_sizes, prefix_lens, self.group, self.kv_heads, prefix_tile,
                           own_tile, tail)

    def plan(self, seq_qlen, group_sizes, prefix_lens, tail: int = 0,
             page: "int | None" = None) -> SharedPlan:
        """The plan of a step (arguments as ``plan_shared``; ``page``: keys of the cache's pages, which
        not all kernels suit) on the device.  It holds for every step of these requests in which they
        bring the same numbers of tokens."""
        return self.host_plan(seq_qlen, group_sizes, prefix_lens, tail, page).to(
            self._device if self._device is not None else "cuda")

    # ------------------------------------------------------------------ device side
    def run(self, q: torch.Tensor, out: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
            block_table: torch.Tensor, seq_slot: torch.Tensor, seq_pos0: torch.Tensor,
            plan: SharedPlan, status: "torch.Tensor | None" = None, buffer=None) -> None:
        """q: a row a token, [heads * d] query features at its front (row stride free), requests in
        the plan's order (``plan``: of any layer with as many heads and kv heads); out [tokens, heads * d]
        (row stride free); keys and values [pages, kv_heads, page, d], this step's tokens' among them;
        ``block_table`` [slots, max pages] int32.
        ``seq_slot`` int32: each request's row of the table; the first of a group has the pages of
        the prefix, all have those of their own keys.  ``seq_pos0`` int32: position of each request's
        first token, not before the prefix's end.  A token sees the keys up to its own position; a
        key without a page is not seen and sets ``status`` (None: what ``ops.take_status`` reads) to 2; a
        bounded wait that ran out sets it to 3.  ``buffer(name, shape, dtype)``: where the partial results
        lie during the call (None: fresh memory)."""
        d, heads, kv_heads, tokens = self.head_dim, self.heads, self.kv_heads, plan.tokens
        if plan.group != self.group or plan.kv_heads != kv_heads:
            raise ValueError(f"shared prefix: the plan is one for {plan.kv_heads} kv heads of {plan.group} "
                             f"query heads each, the layer has {kv_heads} of {self.group}")
        _need(q.dim() == out.dim() == 2, "shared prefix: q and out have a row a token of the plan")
        _need(k_pages.dim() == 4, "shared prefix: pages must be [pages, kv_heads, page, head_dim]")
        q_shape, (q_stride, q_one) = q.shape, q.stride()
        out_shape, (out_stride, out_one) = out.shape, out.stride()
        _need(q.dtype == out.dtype == k_pages.dtype == v_pages.dtype == self.dtype,
              "shared prefix: q, out and the pages have the layer's dtype")
        _need(q_one == 1 and out_one == 1 and q_shape[0] == out_shape[0] == tokens
              and q_shape[1] >= out_shape[1] == heads * d
              and (tokens < 2 or (q_stride >= heads * d and out_stride >= heads * d)),
              "shared prefix: q and out have a row a token of the plan, heads * d features each")
        pages, page_heads, page, page_dim = k_pages.shape
        _need(k_pages.is_contiguous() and v_pages.is_contiguous() and k_pages.shape == v_pages.shape
              and page_heads == kv_heads and page_dim == d and page > 0,
              "shared prefix: pages must be [pages, kv_heads, page, head_dim]")
        _need(block_table.dtype == seq_slot.dtype == seq_pos0.dtype == torch.int32
              and block_table.is_contiguous() and seq_slot.is_contiguous() and seq_pos0.is_contiguous(),
              "shared prefix: block_table, seq_slot and seq_pos0 must be contiguous int32 tensors")
        _need(block_table.dim() == 2 and seq_slot.shape == seq_pos0.shape == plan.seqs.shape[:1],
              "shared prefix: block_table [slots, pages], a slot and a position a request")
        _need(plan.device is not None, "shared prefix: the plan is not on the device yet (plan.to)")
        _on_device(q, out, k_pages, v_pages, block_table, seq_slot, seq_pos0, plan.seqs)
        if tokens == 0:
            return
        status = _status_word(status, q)
        # sums and, behind them, the maximum and the sum of weights of every partial result
        rows = plan.partial_rows * kv_heads
        shape = (rows * (d + 2),)
        partial = (torch.empty(shape, dtype=torch.float32, device=q.device) if buffer is None else
                   buffer("shared_prefix.partial", shape, torch.float32))
        acc = partial.data_ptr()
        ml = acc + 4 * rows * d
        lib = library.load("shared_prefix")
        tag, stream = _tag(self.dtype), _stream()
        q_at, k_at, v_at = q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr()
        # what a kernel copies in pieces has to lie so; the next one in this list takes it otherwise, and
        # what a plan of another type or head size has for kernels that this layer does not have
        pages_fit = not (k_at % 16 or v_at % 16)
        rows_fit = pages_fit and self.dtype == torch.float32 and d % 4 == 0
        aligned = pages_fit and self.tensor_cores and not (q_stride % 2 or q_at % 4)
        wide = pages_fit and self.tcgen05_module is not None and not (q_stride % 8 or q_at % 16)
        before = (q_at, q_stride, k_at, v_at, block_table.data_ptr(), block_table.stride(0), pages,
                  seq_slot.data_ptr(), seq_pos0.data_ptr())
        after = (acc, ml, heads, kv_heads, d, page, self.scale, status.data_ptr(), stream)
        last = len(plan.items) - 1
        for i, (name, items) in enumerate(plan.items.items()):
            order = (i > 0) + 2 * (i < last)              # behind another kernel, followed by one
            rows, unit = plan.shapes[name]
            work = (*before, items.data_ptr(), items.shape[0])
            if (name == "tcgen05" and wide and not i
                    and (kernel := library.load(*self.tcgen05_module)).de_shared_tcgen05_page_ok(page)):
                _check(kernel.de_shared_tcgen05(*work, plan.turns, *after),
                       "shared prefix attention (tcgen05)")
            elif name.startswith("f32") and rows_fit:
                _check(library.load("shared_prefix_f32").de_shared_f32(*work, rows, order, *after),
                       "shared prefix attention (float32)")
            elif name in ("warp", "tcgen05") and aligned:
                _check(library.load(*self.mma_module).de_shared_mma(*work, rows, order, *after),
                       "shared prefix attention (mma)")
            else:
                _check(lib.de_shared_rows(tag, *work, rows, unit, order, *after),
                       "shared prefix attention")
        _check(lib.de_shared_merge(tag, out.data_ptr(), out_stride, plan.token_seq.data_ptr(),
                                   plan.seqs.data_ptr(), acc, ml, plan.most_parts, tokens, heads,
                                   kv_heads, d, stream), "shared prefix merge")
