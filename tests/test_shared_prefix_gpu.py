"""Attention whose requests share prefixes against the definition in 64 bits: a request's keys are one
sequence, whoever shares them.  Free pages, and the places of a page behind a request's last key, hold
NaN."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _layer(*args):
    from distengine_b200.kernels.shared_prefix import SharedPrefixAttention
    return SharedPrefixAttention(*args, torch.device(DEV))


class Case:
    """Groups of requests, [(prefix, [(own keys, new tokens), ...]), ...], in scattered pages."""

    def __init__(self, groups, heads, kv_heads, d, page, dtype, seed=0, spread=1.0, poison=True):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.d, self.page, self.dtype = heads, kv_heads, d, page, dtype
        self.sizes = [len(members) for _, members in groups]
        self.prefix = [p for p, _ in groups]
        self.qlen = [n for _, members in groups for _, n in members]
        self.pos0 = [p + own for p, members in groups for own, _ in members]
        tables, used, self.k, self.v = [], 0, [], []
        content = []                            # (request, logical page) -> page, in order
        for p, members in groups:
            kp, vp = (torch.randn(p, kv_heads, d, generator=g).to(dtype) for _ in range(2))
            common = list(range(used, used + p // page))
            used += len(common)
            for own, n in members:
                total = p + own + n
                k, v = (torch.cat((x, torch.randn(own + n, kv_heads, d, generator=g).to(dtype)))
                        for x in (kp, vp))
                more = -(-total // page) - len(common)
                tables.append(common + list(range(used, used + more)))
                used += more
                self.k.append(k), self.v.append(v)
                content.append(tables[-1])
        order = torch.randperm(used + 3, generator=g)
        slots = torch.randperm(len(tables) + 2, generator=g)[: len(tables)]
        width = max([len(t) for t in tables] + [1]) + 1
        self.table = torch.full((len(tables) + 2, width), -1, dtype=torch.int32)
        nan = float("nan") if poison else 0.0
        self.k_pages = torch.full((used + 3, kv_heads, page, d), nan, dtype=dtype)
        self.v_pages = torch.full((used + 3, kv_heads, page, d), nan, dtype=dtype)
        for s, t in enumerate(content):
            for logical, p in enumerate(t):
                at = int(order[p])
                self.table[slots[s], logical] = at
                rows = slice(logical * page, min((logical + 1) * page, self.k[s].shape[0]))
                n = rows.stop - rows.start
                self.k_pages[at, :, :n] = self.k[s][rows].transpose(0, 1)
                self.v_pages[at, :, :n] = self.v[s][rows].transpose(0, 1)
        self.slots = slots.int()
        self.tokens = sum(self.qlen)
        self.scale = d ** -0.5
        self.q = (torch.randn(self.tokens, heads, d, generator=g) * spread).to(dtype)

    def want(self):
        """(results float64 [tokens, heads, d], how far a result in this dtype may be off)."""
        heads, d, rep = self.heads, self.d, self.heads // self.kv_heads
        out = torch.zeros(self.tokens, heads, d, dtype=torch.float64)
        tol = torch.zeros_like(out)
        eps = 2.0 ** -24
        at = 0
        for s, n in enumerate(self.qlen):
            if n == 0:
                continue
            k = self.k[s].double().repeat_interleave(rep, 1).to(DEV)
            v = self.v[s].double().repeat_interleave(rep, 1).to(DEV)
            for t in range(n):
                m = self.pos0[s] + t + 1
                q = self.q[at + t].double().to(DEV)
                score = torch.einsum("hd,jhd->hj", q, k[:m]) * self.scale
                w = torch.softmax(score, 1)
                out[at + t] = torch.einsum("hj,jhd->hd", w, v[:m]).cpu()
                mass = torch.einsum("hj,jhd->hd", w, v[:m].abs()).cpu()
                # scores: d products and sums, on the tensor cores with a sum that may be cut instead
                # of rounded (factor 2); their exponent again two roundings of its size; exp2 2^-21;
                # a sum over m keys in any order, joined from up to 600 ranges; all of it in the
                # numerator and in the denominator
                dots = (torch.einsum("hd,jhd->hj", q.abs(), k[:m].abs()) * self.scale).amax(1).cpu()
                rel = 2 * (d + 4) * eps * dots + 4 * eps * score.abs().amax(1).cpu() + 2.0 ** -21
                rel = 2 * (rel + 2 * (m + 600) * eps)
                tol[at + t] = rel[:, None] * mass
                if self.dtype == torch.bfloat16:      # half a step: of each weight, and of the result
                    tol[at + t] += 2.0 ** -8 * mass + 2.0 ** -8 * out[at + t].abs()
            at += n
        return out, tol + 1e-30

    def run(self, layer=None, plan=None, tail=0, q_pad=0, out_pad=0, status=None, buffer=None):
        layer = layer or _layer(self.dtype, self.heads, self.kv_heads, self.d, self.scale)
        plan = plan or layer.plan(self.qlen, self.sizes, self.prefix, tail)
        width = self.heads * self.d
        q = torch.full((self.tokens + 1, width + q_pad), 9.0, dtype=self.dtype, device=DEV)
        q[: self.tokens, :width] = self.q.view(self.tokens, width).to(DEV)
        out = torch.full((self.tokens + 1, width + out_pad), 77.0, dtype=self.dtype, device=DEV)
        status = torch.zeros(1, dtype=torch.int32, device=DEV) if status is None else status
        layer.run(q[: self.tokens], out[: self.tokens, :width], self.k_pages.to(DEV),
                  self.v_pages.to(DEV), self.table.to(DEV), self.slots.to(DEV),
                  torch.tensor(self.pos0, dtype=torch.int32, device=DEV), plan, status, buffer)
        torch.cuda.synchronize()
        assert bool((out[self.tokens:] == 77.0).all()) and bool((out[:, width:] == 77.0).all())
        self.status = int(status.item())
        return out[: self.tokens, :width].double().cpu().view(self.tokens, self.heads, self.d)

    def check(self, **how):
        got = self.run(**how)
        want, tol = self.want()
        assert self.status == 0
        assert bool(got.isfinite().all())
        off = ((got - want).abs() / tol).max().item() if self.tokens else 0.0
        assert off <= 1.0, f"{off:.2f} times what the roundings allow"
        return got


GROUPS = {
    "beams": [(80, [(5, 1), (0, 1), (17, 1), (30, 1)])],
    "one_key": [(1, [(0, 1), (0, 1)])],
    "no_prefix": [(0, [(0, 1), (40, 1), (99, 1)])],
    "alone": [(100, [(3, 1)]), (64, [(0, 1)])],
    "uneven": [(33, [(0, 1), (7, 1), (2, 1)]), (200, [(1, 1)]), (129, [(150, 1), (0, 1)]),
               (0, [(4, 1)])],
    "portions": [(70, [(5, 3), (0, 1), (9, 20)]), (45, [(2, 7), (0, 33)]), (0, [(0, 5)])],
    "absent": [(50, [(5, 0), (3, 1), (1, 2)]), (60, [(4, 0), (2, 1)]), (64, [(1, 0), (0, 0)])],
    "many": [(300, [(i % 7, 1) for i in range(70)]), (140, [(3 * i, 1) for i in range(40)])],
    "long": [(3001, [(i * 90, 1) for i in range(6)])],
}
HEADS = [(8, 2, 64), (4, 4, 128), (6, 2, 16), (32, 4, 64), (16, 2, 128), (5, 1, 32), (9, 3, 80),
         (2, 1, 256), (8, 8, 64), (40, 2, 128)]
DTYPES = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("groups", sorted(GROUPS))
@pytest.mark.parametrize("heads", HEADS[:4])
@pytest.mark.parametrize("dtype", DTYPES)
def test_groups(groups, heads, dtype):
    Case(GROUPS[groups], *heads, 16, dtype, seed=len(groups)).check(tail=40, q_pad=16)


@pytest.mark.parametrize("heads", HEADS[4:] + [(4, 2, 6), (4, 2, 98), (3, 3, 2)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_head_layouts(heads, dtype):
    Case(GROUPS["uneven"] + GROUPS["portions"], *heads, 16, dtype, seed=3).check()
    Case(GROUPS["many"], *heads, 16, dtype, seed=4).check(tail=500)


@pytest.mark.parametrize("page", [1, 8, 24, 64, 100, 128, 256])
@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_pages(page, heads, dtype):
    Case(GROUPS["uneven"] + GROUPS["beams"] + GROUPS["many"][:1], *heads, page, dtype, seed=page).check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_large_scores(dtype):
    """Rows of odd strides (no 16-byte pieces), and scores far apart."""
    for pad in (1, 3, 8, 200):
        Case(GROUPS["uneven"], 8, 2, 64, 16, dtype, seed=pad).check(q_pad=pad, out_pad=pad)
    Case(GROUPS["many"], 8, 2, 128, 16, dtype, seed=1, spread=20.0).check()
    Case(GROUPS["long"], 8, 1, 64, 16, dtype, seed=2, spread=40.0).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [(16, 4, 64), (32, 8, 128)])
def test_long_prefixes(dtype, heads):
    Case([(9001, [(i * 13, 1) for i in range(20)]), (4097, [(0, 2)] * 3)], *heads, 64, dtype,
         seed=5).check(tail=300)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_plan_holds_from_step_to_step(dtype):
    """The same plan while the requests' own keys grow, well past what it was told to expect."""
    layer = _layer(dtype, 8, 2, 64, 64 ** -0.5)
    plan = layer.plan([1] * 5, [3, 2], [130, 64], tail=4)
    for own in (0, 1, 15, 64, 700):
        Case([(130, [(own, 1), (own + 3, 1), (own, 1)]), (64, [(own, 1), (0, 1)])], 8, 2, 64, 16,
             dtype, seed=own).check(layer=layer, plan=plan)


@pytest.mark.parametrize("made,used", [((torch.float32, 64), (torch.bfloat16, 64)),
                                       ((torch.bfloat16, 64), (torch.float32, 64)),
                                       ((torch.bfloat16, 128), (torch.bfloat16, 32)),
                                       ((torch.bfloat16, 128), (torch.bfloat16, 6)),
                                       ((torch.float32, 64), (torch.float32, 6))])
def test_a_plan_of_another_type_or_head_size(made, used):
    """It names kernels that the layer does not have: others do their work."""
    (dtype, d), groups = used, GROUPS["many"] + GROUPS["portions"]
    case = Case(groups, 8, 2, d, 16, dtype, seed=50)
    layer = _layer(made[0], 8, 2, made[1], 0.1)
    case.check(plan=layer.plan(case.qlen, case.sizes, case.prefix, 100))


@pytest.mark.parametrize("dtype", DTYPES)
def test_sharing_changes_no_request(dtype):
    """A request's result is the same, but for the order of the sums, whoever else is in its group."""
    own = [(i * 5, 1) for i in range(20)]
    shared = Case([(400, own)], 8, 2, 64, 16, dtype, seed=9)
    got = shared.check()
    apart = Case([(0, [(400 + o, n)]) for o, n in own], 8, 2, 64, 16, dtype, seed=9)
    apart.q, apart.k, apart.v = shared.q, shared.k, shared.v
    apart.k_pages, apart.v_pages, apart.table, apart.slots = (
        shared.k_pages, shared.v_pages, shared.table, shared.slots)
    apart.pos0 = shared.pos0
    want, tol = shared.want()
    assert bool(((apart.run() - got).abs() <= 2 * tol).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 2, 128), (4, 2, 40)])
@pytest.mark.parametrize("many", [False, True])
def test_what_is_not_finite(dtype, heads, many):
    """An infinity or NaN reaches the tokens that see its key and no others."""
    groups = [(90, [(3, 1), (8, 9), (0, 1)] + [(1, 1)] * (60 if many else 0)), (64, [(0, 1), (2, 4)]),
              (33, [(0, 1)] * 3)]
    case = Case(groups, *heads, 16, dtype, seed=11)
    inf, nan = float("inf"), float("nan")
    first = [0, len(groups[0][1]), len(groups[0][1]) + 2]
    bad = [(1, 90 + 8 + 4, 0, 3, inf), (1, 90 + 8 + 6, 1, 1, nan), (1, 95, 0, 7, -inf),
           (first[1], 40, 0, 5, inf), (first[1] + 1, 64 + 2 + 1, 1, 2, -inf), (first[2], 2, 1, 0, nan)]
    for s, key, head, feature, value in bad:
        group = max(g for g in range(3) if first[g] <= s)
        shared = key < case.prefix[group]
        for r in range(first[group], first[group] + case.sizes[group]) if shared else [s]:
            case.v[r][key, head, feature] = value
            at = int(case.table[case.slots[r], key // 16])
            case.v_pages[at, head, key % 16, feature] = value
    got = case.run()
    want, tol = case.want()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[want.isinf()], want[want.isinf()])
    fine = want.isfinite()
    assert int((~fine).sum()) > 20 and bool(((got - want).abs()[fine] <= tol[fine]).all())


def test_keys_that_are_not_finite():
    """A score of NaN makes its tokens' results NaN, in float32 and in bfloat16."""
    for dtype in DTYPES:
        case = Case([(70, [(3, 1), (8, 3)]), (40, [(1, 1)] * 2)], 8, 2, 64, 16, dtype, seed=12)
        for r in (0, 1):
            case.k[r][30, 1, 4] = float("nan")
        case.k_pages[int(case.table[case.slots[0], 1]), 1, 14, 4] = float("nan")
        got, (want, tol) = case.run(), case.want()
        assert torch.equal(got.isnan(), want.isnan()) and bool(want.isnan().any())
        fine = want.isfinite()
        assert bool(((got - want).abs()[fine] <= tol[fine]).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 2, 128)])
def test_keys_without_a_page(dtype, heads):
    """They are not seen, and the status says so; a row that sees none gives 0."""
    for many in (1, 70):
        case = Case([(96, [(20, 1)] * (2 * many)), (32, [(0, 1)] * 2)], *heads, 16, dtype, seed=13)
        for row in range(case.table.shape[0]):
            if row in case.slots[: 2 * many].tolist():
                case.table[row, 2] = -1 if row % 2 else 100_000
            else:
                case.table[row] = -1
        for s in range(2 * many):
            keep = torch.cat((torch.arange(32), torch.arange(48, 96 + 21)))
            case.k[s], case.v[s] = case.k[s][keep], case.v[s][keep]
        pos0 = list(case.pos0)
        got = case.run()
        assert case.status == 2
        case.pos0 = [p - 16 for p in pos0]
        for s in (2 * many, 2 * many + 1):
            case.qlen[s] = 0
        want, tol = case.want()
        assert bool(((got - want).abs()[: 2 * many] <= tol[: 2 * many]).all())
        assert bool((got[2 * many:] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_streams_graphs_and_shared_memory(dtype):
    """Two captured calls replayed side by side on two streams, and eager calls on a side stream."""
    layer = _layer(dtype, 8, 2, 64, 64 ** -0.5)
    cases = [Case([(200, [(i, 1) for i in range(12 + 60 * c)])], 8, 2, 64, 16, dtype, seed=20 + c)
             for c in range(2)]
    jobs = []
    for case in cases:
        q = case.q.view(case.tokens, -1).to(DEV)
        args = (q, torch.zeros_like(q), case.k_pages.to(DEV), case.v_pages.to(DEV),
                case.table.to(DEV), case.slots.to(DEV),
                torch.tensor(case.pos0, dtype=torch.int32, device=DEV),
                layer.plan(case.qlen, case.sizes, case.prefix))
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            layer.run(*args)
            eager = args[1].clone()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            layer.run(*args)
        args[1].zero_()
        torch.cuda.synchronize()
        jobs.append((stream, graph, args, eager))
    for _ in range(20):
        for stream, graph, args, _ in jobs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for case, (_, _, args, eager) in zip(cases, jobs):
        assert torch.equal(args[1], eager)
        want, tol = case.want()
        assert bool(((eager.double().cpu().view_as(want) - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_same_bits_every_time(dtype):
    case = Case(GROUPS["many"] + GROUPS["portions"], 8, 2, 64, 16, dtype, seed=30)
    first = case.run()
    for _ in range(5):
        assert torch.equal(case.run(), first)


def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 elements: its last pages are read."""
    free, _ = torch.cuda.mem_get_info()
    kv_heads, page, d = 8, 64, 128
    pages = (1 << 32) // (kv_heads * page * d) + 40
    if free < 3 * pages * kv_heads * page * d * 2:
        pytest.skip("not enough free memory")
    for heads in (8, 64):
        case = Case([(150, [(70, 1)] * 20)], heads, kv_heads, d, page, torch.bfloat16, seed=40)
        n = case.k_pages.shape[0]
        big = [torch.zeros(pages, kv_heads, page, d, dtype=torch.bfloat16, device=DEV)
               for _ in range(2)]
        big[0][-n:], big[1][-n:] = case.k_pages.to(DEV), case.v_pages.to(DEV)
        table = torch.where(case.table >= 0, case.table + (pages - n), -1).to(DEV)
        layer = _layer(torch.bfloat16, heads, kv_heads, d, case.scale)
        q = case.q.view(case.tokens, -1).to(DEV)
        out = torch.zeros_like(q)
        layer.run(q, out, *big, table, case.slots.to(DEV),
                  torch.tensor(case.pos0, dtype=torch.int32, device=DEV),
                  layer.plan(case.qlen, case.sizes, case.prefix))
        want, tol = case.want()
        assert bool(((out.double().cpu().view_as(want) - want).abs() <= tol).all())
        del big


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("d", [64, 128])
def test_pipelines_that_take_turns(page, d):
    """Up to 128 rows a block's two pipelines take the tiles of keys in turn, so a buffer that the one has
    read is filled for the other: which must not take what lay there before for its own, however late
    that one landed.  The same bits every time, whatever the caches hold."""
    case = Case([(12000, [(3, 1)] * 9)], 32, 8, d, page, torch.bfloat16, seed=page + d)
    first = case.check(tail=4)
    for _ in range(8):
        torch.zeros(1 << 28, device=DEV)
        assert torch.equal(case.run(tail=4), first)
