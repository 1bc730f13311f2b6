"""shared_prefix_attention against softmax in 64 bits over a row's prefix and own keys."""
import numpy as np
import pytest
import torch

from tlaloc_b200 import ops

pytestmark = pytest.mark.gpu
F32, BF16, F8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


class Case:
    """Pools whose rows hold NaN but for live positions, tables in random order."""

    def __init__(self, lens, rows, own, *, H=8, Hkv=2, D=128, block=16, pool=BF16, query=BF16, seed=0, starts=None, wide=0, spread=1.0, spare=2):
        rng = np.random.RandomState(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.rows, self.H, self.Hkv, self.D, self.block = list(lens), rows, H, Hkv, D, block
        self.own = [own] * rows if np.isscalar(own) else list(own)
        self.starts = list(starts) if starts is not None else [rows * i // len(self.lens) for i in range(len(self.lens) + 1)]
        counts = [-(-n // block) for n in self.lens + self.own]
        P = sum(counts) + spare
        order = rng.permutation(P).astype(np.int32)
        widths = [max(counts[:len(lens)] + [1]) + wide, max(counts[len(lens):] + [1]) + wide]
        tables = [np.full((len(lens), widths[0]), P + 7, np.int32), np.full((rows, widths[1]), -5, np.int32)]  # what is not live names no page
        live = torch.zeros((P, block), dtype=torch.bool)
        at = 0
        for i, n in enumerate(self.lens + self.own):
            pages = order[at:at + counts[i]]
            at += counts[i]
            (tables[0][i] if i < len(lens) else tables[1][i - len(lens)])[:len(pages)] = pages
            for j, p in enumerate(pages):
                live[p, :min(block, n - j * block)] = True
        dead = ~live.cuda()[:, :, None, None]
        make = lambda s: (torch.randn((P, block, Hkv, D), generator=g, device="cuda") * s).masked_fill(dead, float("nan")).to(pool)  # noqa: E731
        self.kc, self.vc = make(spread), make(1.0)
        self.q = torch.randn((rows, H, D), generator=g, device="cuda").mul(2.0).to(query)
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()  # noqa: E731
        self.prefix_tables, self.tables, self.dl, self.ds, self.do = put(tables[0]), put(tables[1]), put(self.lens), put(self.starts), put(self.own)
        self.scale = D ** -0.5

    def run(self, **kw):
        return ops.shared_prefix_attention(self.q, self.kc, self.vc, self.prefix_tables, self.dl, self.ds, self.tables, self.do, scale=kw.pop("scale", self.scale), **kw)

    def keys(self, cache, row):
        """[n, Hkv, D] in 64 bits."""
        flat = cache.double().view(-1, self.Hkv, self.D)
        out = []
        for g, n in enumerate(self.lens):
            if self.starts[g] <= row < self.starts[g + 1]:
                out.append((self.prefix_tables[g], n))
        out.append((self.tables[row], self.own[row]))
        rows = []
        for table, n in out:
            pos = torch.arange(n, device="cuda")
            rows.append(flat[table[pos // self.block].long() * self.block + pos % self.block])
        return torch.cat(rows)

    def check(self, out, lse=None, rows=None, scale=None):
        """Of a score: D products and sums in f32 (or q in two bf16 parts, 2^-17 of it), 2^-24 each of the sum of sizes; its error moves each weight by as much, twice (the
        weight and the sum); n + 8 roundings of the sums of weighted values, weights in two bf16 parts 2^-17; a bf16 result: weights of one bf16 part
        (2^-8) and its own half step."""
        scale = self.scale if scale is None else scale
        for r in range(self.rows) if rows is None else rows:
            k, v = self.keys(self.kc, r), self.keys(self.vc, r)
            n = k.shape[0]
            if n == 0:
                assert bool((out[r] == 0).all()) and (lse is None or bool((lse[r] == -np.inf).all()))
                continue
            k, v = (t.repeat_interleave(self.H // self.Hkv, 1) for t in (k, v))
            q = self.q[r].double()
            s = torch.einsum("hd,nhd->hn", q, k) * scale
            size = (torch.einsum("hd,nhd->hn", q.abs(), k.abs()) * abs(scale)).amax(1)[:, None]
            p = torch.softmax(s, 1)
            want, bulk = torch.einsum("hn,nhd->hd", p, v), torch.einsum("hn,nhd->hd", p, v.abs())
            move = 2 * size * ((self.D + 2) * 2.0**-24 + 2.0**-17) + (n + 8) * 2.0**-24 + 2.0**-17
            bound = move * bulk
            if out.dtype == BF16:
                bound = bound + 2.0**-8 * bulk + 2.0**-8 * want.abs()
            off = (out[r].double() - want).abs()
            assert bool((off <= bound).all()), (r, (off / bound).max().item())
            if lse is not None:
                gap = (lse[r].double() - torch.logsumexp(s, 1)).abs()
                assert bool((gap <= move[:, 0] + 2.0**-22 * (1 + s.abs().amax(1))).all()), (r, gap.max().item())


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("query", [F32, BF16])
@pytest.mark.parametrize("pool", [F32, BF16, F8])
@pytest.mark.parametrize("D,block", [(64, 16), (128, 16), (80, 24)])
def test_types(D, block, pool, query, out):
    c = Case([333], 9, [1, 2, 15, 16, 17, 31, 32, 33, 100], D=D, block=block, pool=pool, query=query)
    got, lse = c.run(out_dtype=out, return_lse=True)
    c.check(got, lse)


@pytest.mark.parametrize("length", [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000, 4096])
def test_prefix_lengths(length):
    c = Case([length], 5, [0, 1, 20, 3, 0])
    got, lse = c.run(out_dtype=F32, return_lse=True)
    c.check(got, lse)


@pytest.mark.parametrize("rows,H,Hkv", [(1, 1, 1), (1, 32, 8), (3, 8, 8), (7, 10, 2), (16, 32, 4), (33, 32, 8), (64, 16, 2), (65, 16, 2), (100, 24, 8), (127, 8, 1), (128, 64, 8), (160, 16, 1)])
def test_rows_and_heads(rows, H, Hkv):
    c = Case([300], rows, (np.arange(rows) * 13) % 50, H=H, Hkv=Hkv, D=64)
    got, lse = c.run(out_dtype=F32, return_lse=True)
    c.check(got, lse, rows=sorted({0, 1 % rows, rows // 2, rows - 1}))


@pytest.mark.parametrize("D", [1, 7, 32, 64, 72, 96, 128, 192, 200, 256])
def test_head_sizes(D):
    c = Case([150], 4, 9, D=D, H=6, Hkv=3, query=F32)
    c.check(c.run())


@pytest.mark.parametrize("block", [1, 3, 8, 16, 24, 32, 48, 64, 128, 256])
@pytest.mark.parametrize("pool", [BF16, F8])
def test_page_sizes(block, pool):
    c = Case([500, 77], 6, [0, 1, 40, 5, 300, 8], block=block, pool=pool)
    c.check(c.run(out_dtype=F32))


@pytest.mark.parametrize("pool", [BF16, F8])
@pytest.mark.parametrize("lens,rows,starts", [
    ([100, 0, 300], 9, None), ([64] * 9, 9, None), ([700, 3, 1, 129, 128], 40, [0, 1, 1, 30, 35, 40]), ([200, 50], 10, [2, 5, 8]), ([40] * 70, 70, None),
    ([1000, 10], 80, [0, 70, 80]), ([5], 4, [0, 0]), ([513, 512, 511], 96, None)])
def test_groups(lens, rows, starts, pool):
    c = Case(lens, rows, (np.arange(rows) * 7) % 40, starts=starts, pool=pool, Hkv=2, H=8)
    got, lse = c.run(out_dtype=F32, return_lse=True)
    c.check(got, lse)


@pytest.mark.parametrize("rows", [1, 3, 16, 150])
@pytest.mark.parametrize("pool,D", [(F32, 128), (BF16, 80), (F8, 256), (BF16, 128)])
def test_own_lengths_around_slices(pool, D, rows):
    """Own parts in slices of 32 to 256 positions, by how many rows there are."""
    lens = [0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1000]
    c = Case([100], rows, [lens[(5 * r + rows) % len(lens)] for r in range(rows)], H=4, Hkv=2, D=D, pool=pool, query=F32, seed=rows, wide=1024 // 16)
    out, lse = c.run(out_dtype=F32, return_lse=True)
    c.check(out, lse)


def test_long_prefix():
    c = Case([20000], 24, 100, H=16, Hkv=2)
    c.check(c.run(out_dtype=F32), rows=[0, 11, 23])
    c.check(c.run(), rows=[0, 11, 23])


@pytest.mark.parametrize("pool", [F32, BF16, F8])
def test_scores_far_apart(pool):
    """One key outweighs all others, wherever it lies; maxima that keep rising."""
    c = Case([1500], 6, 30, pool=pool, H=4, Hkv=1, D=64)
    flat = c.kc.float().view(-1, 64)
    for r, pos in enumerate([0, 127, 128, 700, 1498, 1499]):
        at = c.prefix_tables[0, pos // 16].long() * 16 + pos % 16
        flat[at] = (c.q[r, 0].float() * 8).clamp(-400, 400)
    pos = torch.arange(0, 1500, 100, device="cuda")
    at = c.prefix_tables[0, pos // 16].long() * 16 + pos % 16
    flat[at] += torch.arange(len(pos), device="cuda")[:, None] * c.q[2, 1].float() * 0.2
    c.kc = flat.view(c.kc.shape).to(pool)
    got, lse = c.run(out_dtype=F32, return_lse=True)
    c.check(got, lse)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.0])
@pytest.mark.parametrize("pool", [F32, BF16])
def test_scales(scale, pool):
    c = Case([200], 4, 10, D=64, pool=pool)
    c.check(c.run(out_dtype=F32, scale=scale), scale=scale)


def test_rows_of_one_table():
    """Several rows of a sequence over one own table, each with its own visible length."""
    c = Case([130], 6, [3, 4, 5, 40, 41, 42])
    c.tables = c.tables[[2, 2, 2, 5, 5, 5]][[0, 3]].contiguous()
    c.kc, c.vc = c.kc.nan_to_num(0.5), c.vc.nan_to_num(0.25)
    out = c.run(out_dtype=F32)
    c.tables = c.tables.repeat_interleave(3, 0)
    c.check(out)


def test_values_that_are_not_numbers_reach_their_heads_alone():
    c = Case([200], 3, 10, H=4, Hkv=2)
    page = int(c.prefix_tables[0, 5])
    c.vc[page, 3, 1, 7] = float("nan")
    out = c.run(out_dtype=F32)
    bad = torch.isnan(out)
    assert bool(bad[:, 2:, 7].all()) and int(bad.sum()) == 3 * 2
    c.kc[page, 3, 0, 0] = float("nan")
    bad = torch.isnan(c.run(out_dtype=F32))
    assert bool(bad[:, :2].all())


def test_wide_tables_and_results_left_alone():
    c = Case([90, 33], 8, 12, wide=50)
    rows = torch.full((10, c.H, c.D), 7.0, dtype=BF16, device="cuda")
    c.run(out=rows[1:9])
    c.check(rows[1:9])
    assert bool((rows[0] == 7).all()) and bool((rows[9] == 7).all())


def test_pools_past_two_to_the_31():
    Hkv, D, block = 8, 128, 16
    P = (1 << 31) // (block * Hkv * D) + 40
    kc = torch.zeros((P, block, Hkv, D), dtype=BF16, device="cuda")
    vc = torch.zeros_like(kc)
    kc[P - 30:].normal_(), vc[P - 30:].normal_()
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.randn((3, 16, D), device="cuda").to(BF16)
    far = [P - 1 - i for i in range(30)]
    args = lambda tables, own: (i32([tables]), i32([300]), i32([0, 3]), i32(own), i32([5, 16, 9]))  # noqa: E731
    got = ops.shared_prefix_attention(q, kc, vc, *args(far[:20], [far[20:22], far[22:24], far[24:26]]), scale=0.1)
    small = [29 - i for i in range(30)]
    want = ops.shared_prefix_attention(q, kc[P - 30:].contiguous(), vc[P - 30:].contiguous(), *args(small[:20], [small[20:22], small[22:24], small[24:26]]), scale=0.1)
    assert torch.equal(got, want)


def test_the_same_result_every_time_and_in_a_graph():
    c = Case([1000, 37], 40, (np.arange(40) * 5) % 60)
    scratch = ops.shared_prefix_scratch(c.q, c.kc, c.prefix_tables, c.tables)
    out = torch.empty_like(c.q)
    first = c.run(scratch=scratch, out=out).clone()
    scratch.fill_(float("nan"))
    assert torch.equal(first, c.run())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(scratch=scratch, out=out)
    out.zero_(), scratch.fill_(float("nan"))
    graph.replay()
    assert torch.equal(first, out)
    # lengths and row ranges are read from the device: a replay follows them
    c.lens, c.starts, c.own = [640, 20], [0, 3, 40], [max(0, n - 3) for n in c.own]
    c.dl.copy_(torch.tensor(c.lens)), c.ds.copy_(torch.tensor(c.starts)), c.do.copy_(torch.tensor(c.own))
    graph.replay()
    c.check(out)


def test_two_streams_with_workspaces_of_their_own():
    cases = [Case([2000], 20, 30, seed=i) for i in range(2)]
    want = [c.run() for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(3):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(c.run())
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want[i % 2])


def test_without_a_prefix_it_is_paged_attention():
    c = Case([0], 12, (np.arange(12) * 11) % 90, query=F32)
    want = ops.paged_attention(c.q, c.kc, c.vc, c.tables, c.do, scale=c.scale)
    assert (c.run() - want).abs().max().item() <= 2.0**-20 * want.abs().max().item()
