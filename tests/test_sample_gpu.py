"""sample against its definition in 64 bits: the same token in every row."""
import numpy as np
import pytest
import torch

from tlaloc_b200 import ops

pytestmark = pytest.mark.gpu


def reference(x, u, t, k, p, m):
    """The token of one row, from the definition; x float64 with -inf for NaN."""
    n = len(x)
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if not t > 0 or top == -np.inf:
        return int(np.argmax(x))
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, 0.0 if top == np.inf else np.exp((x - top) / t))
    w = np.where(x == -np.inf, 0.0, w)
    order = np.lexsort((np.arange(n), -x))
    if 0 < k < n:
        order = order[:k]
    if p < 1:
        sums = np.cumsum(w[order])
        keep = 1 + int(np.count_nonzero(sums[:-1] < max(p, 0.0) * sums[-1]))
        order = order[:keep]
    if m > 0:
        order = order[w[order] >= min(m, 1.0)]
    order = np.sort(order[w[order] > 0])
    sums = np.cumsum(w[order])
    u = 0.0 if not u > 0 else min(u, 1.0)
    return int(order[min(int(np.searchsorted(sums, u * sums[-1], side="right")), len(order) - 1)])


def check(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    rows = logits.shape[0]
    got = ops.sample(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p).tolist()
    host = lambda s: s.double().tolist() if isinstance(s, torch.Tensor) else [float(np.float32(s))] * rows  # noqa: E731
    settings = list(zip(host(temperature), [int(k) for k in host(top_k)], host(top_p), host(min_p)))
    x = logits.double().cpu().numpy()
    want = [reference(x[r], float(u[r]), *settings[r]) for r in range(rows)]
    assert got == want, [(r, got[r], want[r], settings[r], float(u[r])) for r in range(rows) if got[r] != want[r]][:5]


def rows_of(rows, n, seed=0, spread=3.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((rows, n), generator=g, device="cuda") * spread).to(dtype), torch.rand((rows,), generator=g, device="cuda")


SIZES = [1, 2, 31, 32, 33, 100, 1000, 1024, 1025, 4099, 16384, 16385, 32768, 50257, 65537, 128256, 262144, 600001]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", SIZES)
def test_sizes(n, dtype):
    x, u = rows_of(5, n, seed=n, dtype=dtype)
    check(x, u)
    check(x, u, temperature=0.7, top_k=20, top_p=0.9, min_p=0.02)
    check(x, u, top_p=0.99)


@pytest.mark.parametrize("setting", [dict(top_k=1), dict(top_k=2), dict(top_k=50), dict(top_k=999), dict(top_k=5000), dict(top_p=0.0), dict(top_p=1e-6), dict(top_p=0.5),
                                     dict(top_p=0.999), dict(top_p=0.9999999), dict(min_p=0.05), dict(min_p=1.0), dict(min_p=5.0), dict(temperature=0.05),
                                     dict(temperature=1e-20), dict(temperature=50.0), dict(temperature=float("inf")), dict(temperature=0.0), dict(temperature=-1.0),
                                     dict(top_k=40, top_p=0.8), dict(top_k=3000, top_p=0.95, temperature=2.0), dict(top_k=7, min_p=0.5), dict(top_p=0.9, min_p=0.3),
                                     dict(top_k=-4, top_p=2.0, min_p=-1.0), dict(top_p=0.7, temperature=10.0), dict(top_k=20000, top_p=0.97, temperature=3.0)])
@pytest.mark.parametrize("spread", [0.0, 0.3, 3.0, 30.0])
def test_settings(setting, spread):
    x, u = rows_of(24, 32000, seed=3, spread=spread)
    check(x, u, **setting)


def test_settings_of_each_row():
    x, u = rows_of(200, 5000, seed=4)
    rng = np.random.RandomState(1)
    put = lambda a, t: torch.from_numpy(np.asarray(a)).cuda().to(t)  # noqa: E731
    check(x, u, temperature=put(rng.choice([0.0, 0.5, 1.0, 1.7], 200), torch.float32), top_k=put(rng.choice([0, 1, 5, 64, 700], 200), torch.int32),
          top_p=put(rng.choice([0.1, 0.6, 0.95, 1.0], 200), torch.float32), min_p=put(rng.choice([0.0, 0.01, 0.2], 200), torch.float32))


@pytest.mark.parametrize("n", [40, 5000, 40000])
@pytest.mark.parametrize("setting", [dict(), dict(top_k=3), dict(top_k=1000), dict(top_p=0.5), dict(top_k=17, top_p=0.5), dict(min_p=0.9), dict(top_p=0.25, top_k=8)])
def test_equal_values_rank_by_index(n, setting):
    g = torch.Generator(device="cuda").manual_seed(n)
    u = torch.rand((16,), generator=g, device="cuda")
    check(torch.zeros((16, n), device="cuda"), u, **setting)
    few = torch.randint(0, 3, (16, n), generator=g, device="cuda").float()
    few = torch.where(few == 0, -0.0, few - 1)  # -0, 0 and 1: the first two are equal
    check(few, u, **setting)


@pytest.mark.parametrize("setting", [dict(), dict(top_k=5), dict(top_p=0.5), dict(min_p=0.1), dict(top_k=9, top_p=0.7, min_p=0.01), dict(temperature=0.0)])
def test_masked_infinite_and_missing_values(setting):
    x, u = rows_of(12, 3000, seed=6)
    inf = float("inf")
    x[0] = -inf
    x[1] = float("nan")
    x[2, :-1] = -inf
    x[3, 1:] = -inf
    x[4, ::2] = -inf
    x[5, 1::3] = float("nan")
    x[6, 100] = inf
    x[7, 100::500] = inf
    x[8, :] = -inf
    x[8, 17::400] = 1.0
    x[9] = torch.finfo(torch.float32).min
    x[10, 5:] = torch.finfo(torch.float32).min
    x[11, 3] = torch.finfo(torch.float32).max
    check(x, u, **setting)


@pytest.mark.parametrize("n", [4000, 40000])
@pytest.mark.parametrize("setting", [dict(), dict(top_k=700), dict(top_k=3000), dict(top_p=0.5), dict(top_k=2000, top_p=0.7), dict(min_p=0.1), dict(temperature=float("inf"), top_p=0.9)])
def test_many_infinities(setting, n):
    """More of them than one CTA ranks, beside values that then weigh nothing."""
    x, u = rows_of(4, n, seed=n)
    x[0, ::3] = float("inf")
    x[1, 5:] = float("inf")
    x[2] = float("inf")
    x[3, 1::2] = torch.finfo(torch.float32).max
    check(x, u, **setting)


@pytest.mark.parametrize("setting", [dict(), dict(top_k=5), dict(top_p=0.5), dict(temperature=1e30), dict(temperature=1e-30)])
def test_random_numbers_at_their_ends(setting):
    x, _ = rows_of(8, 1000, seed=7)
    u = torch.tensor([0.0, 1.0 - 2.0**-24, 1.0, 2.0, -1.0, float("nan"), float("inf"), 1e-30], device="cuda")
    check(x, u, **setting)


@pytest.mark.parametrize("rows", [0, 1, 2, 17, 148, 149, 300, 1000])
def test_row_counts(rows):
    x, u = rows_of(rows, 2000, seed=rows)
    if rows == 0:
        assert ops.sample(x, u).shape == (0,)
    else:
        check(x, u, top_k=30, top_p=0.9)


@pytest.mark.parametrize("top_k", [600, 1000, 5000])
@pytest.mark.parametrize("top_p", [0.5, 0.95, 0.999])
def test_few_tokens_above_many(top_p, top_k):
    """Rows whose first tokens outweigh thousands of others, cut deep among those."""
    x, u = rows_of(16, 32768, seed=5, spread=2.0)
    x[:, 100:108] += 12.0
    check(x, u, top_k=top_k, top_p=top_p)
    check(x, u, top_p=top_p, temperature=1.4)


@pytest.mark.parametrize("n", [4099, 50257, 128256])
@pytest.mark.parametrize("spread", [0.02, 0.3, 1.0])
@pytest.mark.parametrize("step", [None, 0.001, 0.05])
def test_flat_rows(spread, step, n):
    """Edges among thousands of values that lie close together, or are equal."""
    x, u = rows_of(12, n, seed=n, spread=spread)
    if step is not None:
        x = (x / step).round() * step
    p = torch.tensor([0.0, 0.01, 0.1, 0.3, 0.5, 0.7, 0.9, 0.97, 0.99, 0.999, 0.9999, 0.99999], device="cuda")
    k = torch.tensor([600, 1000, n // 8, n // 4, n // 2, n // 2 + 1, n * 3 // 4, n - 700, n - 1, n, 0, 3000], dtype=torch.int32, device="cuda")
    check(x, u, top_p=p)
    check(x, u, top_k=k)
    check(x, u, top_p=p, top_k=k.flip(0), min_p=0.5)
    check(x, u, top_p=p, top_k=k, temperature=0.3)


@pytest.mark.parametrize("share", [0.9906, 0.9914, 0.9922, 0.9999, 1.0 - 2.0**-24])
def test_values_at_the_ends_of_what_masses_are_guessed_by(share):
    """Two million values just below borders of a 8192nd of an octave, an edge among the scattered ones behind them."""
    part = np.log(2.0) / 8192
    x = np.concatenate([-np.repeat(np.arange(400) * part * (1 + 1e-6), 5000), -(400 + 112 * np.random.RandomState(1).rand(33600)) * part, [-30.0]])
    x = torch.from_numpy(np.random.RandomState(2).permutation(x)).float().cuda().repeat(2, 1)
    check(x, torch.tensor([0.25, 1 - 2.0**-24], device="cuda"), top_p=share)


def test_borders_fall_where_64_bits_have_them():
    """Flat rows over the largest vocabulary: a border between tokens every 4e-6, so that sums of f32 would miss many draws."""
    x, u = rows_of(256, 262144, seed=8, spread=0.5)
    check(x, u)
    check(x, u, top_p=0.97)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lead,ld", [(0, 1003), (1, 1001), (3, 1024)])
def test_rows_of_a_wider_matrix(dtype, lead, ld):
    wide = torch.full((7, ld + lead), 50.0, dtype=dtype, device="cuda")
    x = wide[:, lead:lead + 1000]
    x.normal_()
    check(x, torch.rand((7,), device="cuda"), top_k=50, top_p=0.9)


def test_greedy_is_argmax():
    x, u = rows_of(30, 7777, seed=9, dtype=torch.float32)
    assert torch.equal(ops.sample(x, u, temperature=0.0), ops.argmax(x))


def test_a_captured_call_replays():
    x, u = rows_of(9, 30000, seed=10)
    out = torch.empty((9,), dtype=torch.int32, device="cuda")
    ops.sample(x, u, top_p=0.9, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample(x, u, top_p=0.9, out=out)
    x.copy_(rows_of(9, 30000, seed=11)[0]), u.uniform_()
    graph.replay()
    assert torch.equal(out, ops.sample(x, u, top_p=0.9))


def test_draws_follow_the_distribution():
    """20000 draws of one row: counts within six standard deviations of what they should be."""
    x = torch.log(torch.tensor([[0.5, 0.2, 0.15, 0.1, 0.05]], device="cuda")).repeat(20000, 1)
    counts = torch.bincount(ops.sample(x, torch.rand((20000,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))).long(), minlength=5).double().cpu()
    p = torch.tensor([0.5, 0.2, 0.15, 0.1, 0.05], dtype=torch.float64)
    assert bool(((counts - 20000 * p).abs() <= 6 * (20000 * p * (1 - p)).sqrt()).all())
