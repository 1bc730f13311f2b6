"""norm_rope_kv_write against its definition in 64 bits: norms, both pair layouts, rotations of part of the head, every pairing of types, padding slots, strided rows."""
import numpy as np
import pytest
import torch

from tlaloc_b200 import ops
from tlaloc_b200.rotary import Rotation, YarnScaling, pair_tables

pytestmark = pytest.mark.gpu
F32, BF16, F8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


def reference(x, gain, eps, cos, sin, interleaved):
    """(value, size of what was added up for it) in 64 bits; x [T, heads, hd], cos and sin [T, pairs]."""
    y = x.double()
    if gain is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * gain.double()
    size = y.abs()
    pairs = cos.shape[1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    out, big = y.clone(), size.clone()
    for i in range(pairs):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
        out[..., a] = y[..., a] * c[..., i] - y[..., b] * s[..., i]
        out[..., b] = y[..., b] * c[..., i] + y[..., a] * s[..., i]
        big[..., a] = size[..., a] * c[..., i].abs() + size[..., b] * s[..., i].abs()
        big[..., b] = size[..., b] * c[..., i].abs() + size[..., a] * s[..., i].abs()
    return out, big


def check(got, want, size, hd, normed):
    """f32 arithmetic: three roundings of a rotation, and with a norm hd of its sum (halved by the root) and five more, each 2^-24 of what is added up; then one rounding to
    the type, at most half a step of it (an e4m3 step is 2^-9 at least)."""
    half = {F32: 2.0**-24, BF16: 2.0**-8, F8: 2.0**-4}[got.dtype]
    slack = (3 + (hd / 2 + 5 if normed else 0)) * 2.0**-24 * size
    if got.dtype == F8:
        want = want.clamp(-448, 448)
    off = (got.double() - want).abs()
    bound = slack * (1 + half) + half * want.abs() + (2.0**-10 if got.dtype == F8 else 0.0)
    assert bool((off <= bound).all()), (off - bound).max().item()


def run(T, H, Hkv, hd, pairs, *, interleaved=False, norm=True, x=F32, pool=BF16, q_dtype=BF16, block=16, seed=0, first=0, lead=0, spare=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = dict(device="cuda")
    rows = (torch.randn((T, lead + (H + 2 * Hkv) * hd), generator=g, **dev) * 3).to(x)
    cut = lambda a, n: rows[:, lead + a * hd:lead + (a + n) * hd].unflatten(1, (n, hd))  # noqa: E731
    q, k, v = cut(0, H), cut(H, Hkv), cut(H + Hkv, Hkv)
    gains = [1 + 0.2 * torch.randn((hd,), generator=g, **dev) for _ in range(2)] if norm else [None, None]
    cos, sin = (torch.from_numpy(t).cuda() for t in pair_tables(Rotation(2 * pairs, 10000.0, YarnScaling(4.0, 64.0, 32.0, 1.0)), 200))
    positions = (torch.arange(T, device="cuda") * 7 + first) % 200
    P = -(-T // block) + spare
    slots = torch.randperm(P * block, generator=g, **dev)[:T].int()
    slots[::5] = -1  # padding rows
    if T > 3:
        slots[3] = P * block + 2  # past the pool
    kc, vc = (torch.full((P, block, Hkv, hd), 9.0, **dev).to(pool) for _ in range(2))
    out = ops.norm_rope_kv_write(q, k, v, positions.int(), cos, sin, slots, kc, vc, q_gain=gains[0], k_gain=gains[1], eps=1e-5, interleaved=interleaved, q_dtype=q_dtype)
    c, s = cos[positions], sin[positions]
    check(out, *reference(q, gains[0], 1e-5, c, s, interleaved), hd, norm)
    want_k, size_k = reference(k, gains[1], 1e-5, c, s, interleaved)
    keep = (slots >= 0) & (slots < P * block)
    at = slots[keep].long()
    as_bytes = lambda c: c.view(torch.uint8).reshape(P * block, Hkv, -1)  # noqa: E731
    pick = lambda c: as_bytes(c)[at].contiguous().view(c.dtype).reshape(-1, Hkv, hd)  # noqa: E731
    check(pick(kc), want_k[keep], size_k[keep], hd, norm)
    check(pick(vc), v[keep].double(), torch.zeros_like(v[keep].double()), hd, False)
    untouched = torch.ones((P * block,), dtype=torch.bool, device="cuda")
    untouched[at] = False
    nine = torch.full((1,), 9.0, device="cuda").to(pool)
    for cache in (kc, vc):  # rows that no slot names stay as they were
        assert bool((as_bytes(cache)[untouched] == nine.view(torch.uint8).repeat(hd)).all())
    return out


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hd,pairs", [(2, 1), (3, 1), (32, 16), (64, 32), (64, 8), (80, 24), (96, 48), (96, 13), (128, 64), (128, 32), (128, 0), (136, 68), (192, 32), (256, 128), (256, 32), (320, 160)])
def test_heads_and_rotated_parts(hd, pairs, interleaved):
    run(37, 6, 2, hd, pairs, interleaved=interleaved)
    run(9, 4, 4, hd, pairs, interleaved=interleaved, norm=False, x=BF16, pool=F32, q_dtype=F32)


@pytest.mark.parametrize("x", [F32, BF16])
@pytest.mark.parametrize("pool", [F32, BF16, F8])
@pytest.mark.parametrize("q_dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_types(x, pool, q_dtype, interleaved):
    run(21, 8, 2, 128, 64, x=x, pool=pool, q_dtype=q_dtype, interleaved=interleaved)
    run(21, 5, 5, 64, 16, x=x, pool=pool, q_dtype=q_dtype, interleaved=interleaved, norm=False)


@pytest.mark.parametrize("T", [0, 1, 2, 7, 128, 1000, 2500])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (32, 8), (20, 5), (64, 8)])
def test_tokens(T, H, Hkv):
    run(max(T, 0), H, Hkv, 128, 64) if T else ops.norm_rope_kv_write(
        *(torch.empty((0, n, 8), device="cuda") for n in (H, Hkv, Hkv)), *(torch.empty((0,), dtype=torch.int32, device="cuda") if i in (0, 3) else torch.ones((4, 4), device="cuda")
                                                                           for i in range(4)), *(torch.zeros((2, 4, Hkv, 8), device="cuda") for _ in range(2)))


@pytest.mark.parametrize("lead", [1, 2, 4, 8])
@pytest.mark.parametrize("x", [F32, BF16])
def test_rows_off_16_bytes(lead, x):
    run(33, 6, 3, 64, 32, lead=lead, x=x)


def test_positions_are_clamped():
    q, k, v = (torch.randn((2, 1, 8), device="cuda") for _ in range(3))
    cos, sin = torch.randn((5, 4), device="cuda"), torch.randn((5, 4), device="cuda")
    pools = lambda: [torch.zeros((1, 4, 1, 8), device="cuda") for _ in range(2)]  # noqa: E731
    slots = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    far = ops.norm_rope_kv_write(q, k, v, torch.tensor([-3, 99], dtype=torch.int32, device="cuda"), cos, sin, slots, *pools(), q_dtype=F32)
    ends = ops.norm_rope_kv_write(q, k, v, torch.tensor([0, 4], dtype=torch.int32, device="cuda"), cos, sin, slots, *pools(), q_dtype=F32)
    assert torch.equal(far, ends)


def test_a_pool_row_past_two_to_the_31():
    hkv, hd, block = 8, 128, 16
    P = (1 << 31) // (block * hkv * hd) + 5
    kc = torch.empty((P, block, hkv, hd), dtype=BF16, device="cuda")
    vc = torch.empty_like(kc)
    q, k, v = (torch.randn((1, n, hd), device="cuda") for n in (8, hkv, hkv))
    last = P * block - 1
    ops.norm_rope_kv_write(q, k, v, torch.zeros((1,), dtype=torch.int32, device="cuda"), *(torch.ones((1, 1), device="cuda") * x for x in (1, 0)),
                           torch.tensor([last], dtype=torch.int32, device="cuda"), kc, vc)
    assert torch.equal(kc.view(-1, hkv, hd)[last], k[0].to(BF16)) and torch.equal(vc.view(-1, hkv, hd)[last], v[0].to(BF16))


def test_special_values_stay_in_their_head():
    q, k, v = (torch.randn((3, 4, 64), device="cuda") for _ in range(3))
    q[0, 1, 5], k[1, 2, 3], v[2, 0, 0], v[2, 1, 7] = float("nan"), float("inf"), float("nan"), 1e9
    cos, sin = (torch.from_numpy(t).cuda() for t in pair_tables(Rotation(64, 10000.0), 8))
    ones = torch.ones((64,), device="cuda")
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    kc, vc = (torch.zeros((1, 4, 4, 64), device="cuda").to(F8) for _ in range(2))
    out = ops.norm_rope_kv_write(q, k, v, i32(1, 2, 3), cos, sin, i32(0, 1, 2), kc, vc, q_gain=ones, k_gain=ones, q_dtype=F32)
    bad = torch.isnan(out).any(-1)
    assert bad[0, 1] and int(bad.sum()) == 1
    bad = torch.isnan(kc.float()).any(-1)[0]
    assert bad[1, 2] and int(bad.sum()) == 1
    assert torch.isnan(vc.float())[0, 2, 0, 0] and int(torch.isnan(vc.float()).sum()) == 1 and vc.float()[0, 2, 1, 7] == 448.0


def test_parity_mode_sums_in_order():
    q, k, v = (torch.randn((2, n, 128), device="cuda") for n in (2, 1, 1))
    gain = torch.rand((128,), device="cuda")
    cos, sin = torch.ones((1, 1), device="cuda"), torch.zeros((1, 1), device="cuda")
    at = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    before = ops.set_order_faithful(True)
    try:
        out = ops.norm_rope_kv_write(q, k, v, at * 0, cos, sin, at, *(torch.zeros((1, 2, 1, 128), device="cuda") for _ in range(2)), q_gain=gain, k_gain=gain, eps=1e-5, q_dtype=F32)
        want = ops.rmsnorm(q.view(4, 128), gain, 1e-5)
    finally:
        ops.set_order_faithful(before)
    assert torch.equal(out.view(4, 128), want)


def test_a_captured_call_replays():
    T, H, Hkv, hd = 5, 4, 2, 64
    q, k, v = (torch.randn((T, n, hd), device="cuda") for n in (H, Hkv, Hkv))
    cos, sin = (torch.from_numpy(t).cuda() for t in pair_tables(Rotation(hd, 10000.0), 64))
    at = torch.arange(T, dtype=torch.int32, device="cuda")
    kc, vc = (torch.zeros((2, 16, Hkv, hd), dtype=BF16, device="cuda") for _ in range(2))
    out = torch.empty((T, H, hd), dtype=BF16, device="cuda")
    call = lambda: ops.norm_rope_kv_write(q, k, v, at, cos, sin, at, kc, vc, q_out=out)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    q.normal_(), k.normal_(), v.normal_(), at.add_(3), kc.zero_(), vc.zero_()
    graph.replay()
    replayed = out.clone(), kc.clone(), vc.clone()
    kc.zero_(), vc.zero_()
    call()
    for a, b in zip(replayed, (out, kc, vc)):
        assert torch.equal(a, b)
