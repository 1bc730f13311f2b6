"""What norm_rope_kv_write, shared_prefix_attention and sample refuse, in Python and at the C entries: nothing here launches a kernel."""
import contextlib

import pytest
import torch

from tlaloc_b200 import _native as N
from tlaloc_b200 import ops

I32, F32, BF16 = torch.int32, torch.float32, torch.bfloat16


@pytest.fixture
def calls(monkeypatch):
    """The C functions that were called; tensors on the host count as on a device 0 that is current."""
    seen = []

    class Library:
        def __getattr__(self, name):
            return lambda *args: seen.append((name, args)) or 0

    monkeypatch.setattr(ops.N, "lib", lambda: Library())
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 1000 + device, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    return seen


class OnDevice(torch.Tensor):
    is_cuda = True
    where = 0

    def get_device(self):
        return self.where


def dev(t, where=0):
    t = t.as_subclass(OnDevice)
    t.where = where
    return t


def append(**change):
    T, H, Hkv, hd = 3, 4, 2, 8
    a = dict(q=torch.zeros(T, H, hd), k=torch.zeros(T, Hkv, hd), v=torch.zeros(T, Hkv, hd), positions=torch.zeros(T, dtype=I32), cos=torch.zeros(5, 4), sin=torch.zeros(5, 4),
             slot_mapping=torch.zeros(T, dtype=I32), key_cache=torch.zeros(2, 4, Hkv, hd), value_cache=torch.zeros(2, 4, Hkv, hd), q_gain=torch.ones(hd), k_gain=torch.ones(hd))
    a["q_out"] = torch.zeros(T, H, hd)
    a.update(change)
    a = {n: dev(t) if isinstance(t, torch.Tensor) and not isinstance(t, OnDevice) else t for n, t in a.items()}
    gains = {n: a.pop(n) for n in ("q_gain", "k_gain", "q_out")}
    return ops.norm_rope_kv_write(*a.values(), **gains)


def prefix(**change):
    R, H, Hkv, D, G = 4, 4, 2, 8, 2
    a = dict(query=torch.zeros(R, H, D), key_cache=torch.zeros(3, 4, Hkv, D), value_cache=torch.zeros(3, 4, Hkv, D), prefix_tables=torch.zeros(G, 2, dtype=I32),
             prefix_lens=torch.zeros(G, dtype=I32), row_starts=torch.zeros(G + 1, dtype=I32), block_tables=torch.zeros(R, 2, dtype=I32), seq_lens=torch.zeros(R, dtype=I32))
    keep = dict(out=torch.zeros(R, H, D), scratch=torch.zeros(16))
    keep.update({n: change.pop(n) for n in list(change) if n in keep})
    a.update(change)
    wrap = lambda t: dev(t) if isinstance(t, torch.Tensor) and not isinstance(t, OnDevice) else t  # noqa: E731
    return ops.shared_prefix_attention(*map(wrap, a.values()), scale=1.0, **{n: wrap(t) for n, t in keep.items()})


def draw(logits=None, uniforms=None, **settings):
    logits, uniforms = torch.zeros(3, 7) if logits is None else logits, torch.zeros(3) if uniforms is None else uniforms
    wrap = lambda t: dev(t) if isinstance(t, torch.Tensor) and not isinstance(t, OnDevice) else t  # noqa: E731
    return ops.sample(wrap(logits), wrap(uniforms), out=dev(torch.zeros(3, dtype=I32)), **{n: wrap(t) for n, t in settings.items()})


def test_calls_that_fit_are_made(calls):
    append(), prefix(), draw(temperature=torch.ones(3), top_k=5)
    append(q_gain=None, k_gain=None)
    assert [name for name, _ in calls] == ["tlaloc_b200_norm_rope_kv_write", "tlaloc_b200_shared_prefix_attention", "tlaloc_b200_sample", "tlaloc_b200_norm_rope_kv_write"]
    assert all(args[-1] == 1000 for _, args in calls)  # the stream of the operands' device


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(3, 32)), dict(q=torch.zeros(2, 4, 8)), dict(k=torch.zeros(3, 2, 6)), dict(v=torch.zeros(3, 1, 8)), dict(q=torch.zeros(3, 4, 16)[:, :, ::2]),
    dict(q=torch.zeros(3, 8, 8)[:, ::2]), dict(q=torch.zeros(3, 4, 8, dtype=BF16)), dict(positions=torch.zeros(3, dtype=torch.int64)), dict(positions=torch.zeros(2, dtype=I32)),
    dict(slot_mapping=torch.zeros(4, dtype=I32)), dict(cos=torch.zeros(5, 3)), dict(cos=torch.zeros(0, 4), sin=torch.zeros(0, 4)), dict(cos=torch.zeros(5, 4, dtype=BF16)),
    dict(sin=torch.zeros(5, 8)[:, ::2]), dict(q_gain=torch.ones(7)), dict(q_gain=torch.ones(8, dtype=BF16)), dict(key_cache=torch.zeros(2, 4, 3, 8)),
    dict(value_cache=torch.zeros(2, 4, 2, 8, dtype=BF16)), dict(key_cache=torch.zeros(2, 8, 2, 8)[:, ::2]), dict(q_out=torch.zeros(3, 4, 9)), dict(q_out=torch.zeros(3, 4, 8, dtype=I32)),
    dict(slot_mapping=dev(torch.zeros(3, dtype=I32), 1)), dict(k=dev(torch.zeros(3, 2, 8), 1))])
def test_append_refuses(calls, change):
    with pytest.raises((ValueError, TypeError), match="NORM_ROPE_KV_WRITE"):
        append(**change)
    assert calls == []


@pytest.mark.parametrize("change", [
    dict(query=torch.zeros(4, 32)), dict(query=torch.zeros(4, 4, 6)), dict(value_cache=torch.zeros(3, 4, 2, 9)), dict(value_cache=torch.zeros(3, 4, 2, 8, dtype=BF16)),
    dict(prefix_tables=torch.zeros(2, dtype=I32)), dict(prefix_tables=torch.zeros(3, 2, dtype=I32)), dict(prefix_tables=torch.zeros(2, 2, dtype=torch.int64)),
    dict(prefix_lens=torch.zeros(3, dtype=I32)), dict(row_starts=torch.zeros(2, dtype=I32)), dict(row_starts=torch.zeros(3)), dict(seq_lens=torch.zeros(3, dtype=I32)),
    dict(block_tables=torch.zeros(4, 4, dtype=I32)[:, ::2]), dict(out=torch.zeros(4, 4, 9)), dict(out=torch.zeros(4, 4, 8, dtype=torch.float16)), dict(scratch=torch.zeros(4, dtype=BF16)),
    dict(seq_lens=dev(torch.zeros(4, dtype=I32), 1))])
def test_shared_prefix_refuses(calls, change):
    with pytest.raises((ValueError, TypeError), match="SHARED_PREFIX_ATTENTION"):
        prefix(**change)
    assert calls == []


@pytest.mark.parametrize("change", [
    dict(logits=torch.zeros(21)), dict(logits=torch.zeros(3, 0)), dict(logits=torch.zeros(3, 14)[:, ::2]), dict(uniforms=torch.zeros(2)), dict(uniforms=torch.zeros(3, dtype=torch.float64)),
    dict(uniforms=torch.zeros(6)[::2]), dict(temperature=torch.ones(2)), dict(top_k=torch.ones(3)), dict(top_p=torch.ones(3, dtype=torch.float64)), dict(min_p=torch.ones(3, 1)),
    dict(min_p=dev(torch.ones(3), 1))])
def test_sample_refuses(calls, change):
    with pytest.raises((ValueError, TypeError), match="SAMPLE"):
        draw(**change)
    assert calls == []


def test_operands_on_the_host_are_refused(calls):
    with pytest.raises(ValueError):
        ops.sample(torch.zeros(3, 7), torch.zeros(3))
    assert calls == []


def test_a_call_makes_the_device_of_its_operands_current(calls, monkeypatch):
    current = []

    @contextlib.contextmanager
    def device(index):
        current.append(index)
        yield
        current.append(None)

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(ops, "_out", lambda *a: None)
    ops.sample(dev(torch.zeros(3, 7), 5), dev(torch.zeros(3), 5), out=dev(torch.zeros(3, dtype=I32), 5))
    assert current == [5, None] and calls[0][1][-1] == 1005


# ---------------------------------------------------------------- the C entries

P = 1 << 20  # an address that is never read


def at(i):
    return P * (i + 1)


def c_append(**change):
    a = dict(q=at(0), ld_q=32, k=at(1), ld_k=16, v=at(2), ld_v=16, x_dtype=N.F32, q_gain=at(3), k_gain=at(4), eps=1e-6, positions=at(5), cos=at(6), sin=at(7), slots=at(8),
             q_out=at(9), q_out_dtype=N.BF16, kc=at(10), vc=at(11), kv_dtype=N.BF16, T=3, H=4, Hkv=2, hd=8, rot=8, interleaved=0, num_slots=8, max_pos=5)
    a.update(change)
    return N.lib().tlaloc_b200_norm_rope_kv_write(*a.values(), None)


@pytest.mark.parametrize("change,status", [
    (dict(q=None), N.INVALID_ARGUMENT), (dict(slots=None), N.INVALID_ARGUMENT), (dict(cos=None), N.INVALID_ARGUMENT), (dict(vc=None), N.INVALID_ARGUMENT),
    (dict(x_dtype=N.S8), N.INVALID_ARGUMENT), (dict(q_out_dtype=N.F8E4M3FN), N.INVALID_ARGUMENT), (dict(kv_dtype=N.S32), N.INVALID_ARGUMENT), (dict(T=-1), N.INVALID_ARGUMENT),
    (dict(H=0), N.INVALID_ARGUMENT), (dict(hd=0), N.INVALID_ARGUMENT), (dict(rot=7), N.INVALID_ARGUMENT), (dict(rot=10), N.INVALID_ARGUMENT), (dict(rot=-2), N.INVALID_ARGUMENT),
    (dict(q_gain=None), N.INVALID_ARGUMENT), (dict(k_gain=None), N.INVALID_ARGUMENT), (dict(eps=float("nan")), N.INVALID_ARGUMENT), (dict(eps=-1.0), N.INVALID_ARGUMENT),
    (dict(ld_q=31), N.INVALID_ARGUMENT), (dict(ld_v=15), N.INVALID_ARGUMENT), (dict(num_slots=0), N.INVALID_ARGUMENT), (dict(max_pos=0), N.INVALID_ARGUMENT),
    (dict(H=70000, ld_q=70000 * 8), N.UNSUPPORTED), (dict(q_out=at(0)), N.INVALID_ARGUMENT), (dict(q_out=at(0) + 380), N.INVALID_ARGUMENT), (dict(kc=at(1) - 8), N.INVALID_ARGUMENT),
    (dict(vc=at(10)), N.INVALID_ARGUMENT), (dict(T=0), N.OK)])
def test_c_append_refuses(change, status):
    assert c_append(**change) == status
    if status != N.OK:
        assert b"NORM_ROPE_KV_WRITE" in N.lib().tlaloc_b200_last_error()


def c_prefix(**change):
    a = dict(q=at(0), q_dtype=N.BF16, kc=at(1), vc=at(2), kv_dtype=N.BF16, prefix_tables=at(3), prefix_lens=at(4), row_starts=at(5), tables=at(6), lens=at(7), out=at(8), out_dtype=N.BF16,
             lse=None, scratch=at(9), scratch_bytes=1 << 40, R=4, H=4, D=8, P=3, bs=4, Hkv=2, G=2, Mp=2, M=2, Tb=4, scale=1.0)
    a.update(change)
    return N.lib().tlaloc_b200_shared_prefix_attention(*a.values(), None)


@pytest.mark.parametrize("change,status", [
    (dict(q=None), N.INVALID_ARGUMENT), (dict(prefix_lens=None), N.INVALID_ARGUMENT), (dict(row_starts=None), N.INVALID_ARGUMENT), (dict(lens=None), N.INVALID_ARGUMENT),
    (dict(scratch=None), N.INVALID_ARGUMENT), (dict(q_dtype=N.S8), N.INVALID_ARGUMENT), (dict(kv_dtype=N.S8), N.INVALID_ARGUMENT), (dict(out_dtype=N.F8E4M3FN), N.INVALID_ARGUMENT),
    (dict(G=0), N.INVALID_ARGUMENT), (dict(Mp=0), N.INVALID_ARGUMENT), (dict(bs=0), N.INVALID_ARGUMENT), (dict(Mp=1 << 29), N.UNSUPPORTED), (dict(scratch_bytes=64), N.INVALID_ARGUMENT),
    (dict(scratch=at(9) + 16), N.INVALID_ARGUMENT), (dict(R=0), N.INVALID_ARGUMENT), (dict(Hkv=0), N.INVALID_ARGUMENT), (dict(H=5), N.INVALID_ARGUMENT), (dict(D=257), N.UNSUPPORTED), (dict(Tb=3), N.INVALID_ARGUMENT),
    (dict(M=0), N.INVALID_ARGUMENT), (dict(scale=float("nan")), N.INVALID_ARGUMENT), (dict(scale=float("inf")), N.INVALID_ARGUMENT)])
def test_c_shared_prefix_refuses(change, status):
    assert c_prefix(**change) == status
    assert b"SHARED_PREFIX_ATTENTION" in N.lib().tlaloc_b200_last_error()


def test_c_shared_prefix_has_no_parity_mode():
    before = ops.set_order_faithful(True)
    try:
        assert c_prefix() == N.UNSUPPORTED
    finally:
        ops.set_order_faithful(before)


def test_scratch_grows_with_what_it_holds():
    size = N.lib().tlaloc_b200_shared_prefix_scratch_bytes
    base = size(64, 32, 8, 128, 1, 64, 16)
    assert base > 0 and size(128, 32, 8, 128, 1, 64, 16) > base and size(64, 32, 8, 128, 30, 64, 16) > base and size(64, 32, 8, 128, 1, 640, 16) > base
    assert size(0, 32, 8, 128, 1, 64, 16) == size(64, 32, 0, 128, 1, 64, 16) == size(64, 32, 8, 128, 0, 64, 16) == 0


@pytest.mark.parametrize("change", [dict(logits=None), dict(uniforms=None), dict(out=None), dict(dtype=N.S8), dict(rows=-1), dict(n=0), dict(ld=6)])
def test_c_sample_refuses(change):
    a = dict(logits=at(0), ld=7, dtype=N.F32, uniforms=at(1), temperature=None, top_k=None, top_p=None, min_p=None, t=1.0, k=0, p=1.0, m=0.0, out=at(2), rows=3, n=7)
    a.update(change)
    assert N.lib().tlaloc_b200_sample(*a.values(), None) == N.INVALID_ARGUMENT
    assert b"SAMPLE" in N.lib().tlaloc_b200_last_error()
