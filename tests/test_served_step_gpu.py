"""norm_rope_kv_write, shared_prefix_attention and sample together, as a decode step runs them: a step over a toy model against 64 bits, eager and from a CUDA graph;
and sampled generation through the engine."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import latent_oracle as oracle
from tlaloc_b200 import ops
from tlaloc_b200.sampling import Sampling

pytestmark = pytest.mark.gpu
F32, BF16, F8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def draw(x, u, s):
    """The token of one row of logits x in 64 bits for settings s, from the definition."""
    if s.temperature == 0:
        return int(np.argmax(x))
    f32 = lambda a: float(np.float32(a))  # noqa: E731
    w = np.exp((x - x.max()) / f32(s.temperature))
    order = np.lexsort((np.arange(len(x)), -x))
    if 0 < s.top_k < len(x):
        order = order[:s.top_k]
    if s.top_p < 1:
        sums = np.cumsum(w[order])
        order = order[:1 + int(np.count_nonzero(sums[:-1] < f32(s.top_p) * sums[-1]))]
    order = np.sort(order[w[order] >= f32(s.min_p)])
    sums = np.cumsum(w[order])
    return int(order[min(int(np.searchsorted(sums, u * sums[-1], side="right")), len(order) - 1)])


class Toy:
    """One attention layer: x = table[id], q | k | v = x W, attention, logits = attention V.  Rows [0, 2) continue one prompt, rows [2, 5) another."""

    H, HKV, D, BLOCK, VOCAB, WIDTH, PROMPTS, STARTS = 8, 2, 64, 16, 1031, 96, (37, 150), (0, 2, 5)

    def __init__(self, pool, query):
        g = torch.Generator(device="cuda").manual_seed(3)
        rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        H, K, D = self.H, self.HKV, self.D
        self.table, self.w, self.head = rand(self.VOCAB, self.WIDTH), rand(self.WIDTH, (H + 2 * K) * D) / self.WIDTH**0.5, rand(H * D, self.VOCAB) / 8
        self.gains = [1 + 0.2 * rand(D).clamp(-2, 2), 1 + 0.2 * rand(D).clamp(-2, 2)]
        angles = torch.arange(400)[:, None] * 10000.0 ** (-torch.arange(24) / 24.0)[None]
        self.cos, self.sin = angles.cos().float().cuda(), angles.sin().float().cuda()
        self.kc, self.vc = (torch.full((40, self.BLOCK, K, D), float("nan"), device="cuda").to(pool) for _ in range(2))
        self.query = query
        order = torch.randperm(39, generator=torch.Generator().manual_seed(5)).int() + 1
        i32 = lambda a: torch.as_tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        self.prefix_tables, self.tables = i32(order[:20]).view(2, 10), i32(order[20:35]).view(5, 3)
        self.lens, self.starts, self.own = i32(self.PROMPTS), i32(self.STARTS), i32([0] * 5)
        self.row_lens = i32([37, 37, 150, 150, 150])
        self.rows = torch.arange(5, device="cuda")
        self.prompts = [torch.randint(0, self.VOCAB, (n,), generator=g, device="cuda") for n in self.PROMPTS]
        for p, t in zip(self.prompts, self.prefix_tables):
            pos = torch.arange(len(p), device="cuda")
            self.append(p, pos.int(), (t[pos // self.BLOCK] * self.BLOCK + pos % self.BLOCK).int())
        self.ids, self.u, self.next = i32([5, 5, 9, 700, 9]), torch.zeros(5, device="cuda"), i32([0] * 5)
        s = self.settings = [Sampling(0.8, seed=1), Sampling(1.0, 40, 0.9, seed=2), Sampling(0.0), Sampling(1.3, 0, 0.7, 0.01, seed=4), Sampling(1.0, 0, 1.0, 0.2, seed=5)]
        f32 = lambda a: torch.tensor(a, dtype=F32, device="cuda")  # noqa: E731
        self.how = dict(temperature=f32([a.temperature for a in s]), top_k=i32([a.top_k for a in s]), top_p=f32([a.top_p for a in s]), min_p=f32([a.min_p for a in s]))

    def append(self, ids, positions, slots):
        H, K, D = self.H, self.HKV, self.D
        y = self.table[ids.long()] @ self.w
        q, k, v = y[:, :H * D].unflatten(1, (H, D)), y[:, H * D:(H + K) * D].unflatten(1, (K, D)), y[:, (H + K) * D:].unflatten(1, (K, D))
        return ops.norm_rope_kv_write(q, k, v, positions, self.cos, self.sin, slots, self.kc, self.vc, q_gain=self.gains[0], k_gain=self.gains[1], q_dtype=self.query)

    def step(self):
        """Reads ids, u and own; writes logits and next, then advances."""
        slots = (self.tables[self.rows, self.own.long() // self.BLOCK] * self.BLOCK + self.own % self.BLOCK).int()
        q = self.append(self.ids, self.row_lens + self.own, slots)
        self.own += 1
        att = ops.shared_prefix_attention(q, self.kc, self.vc, self.prefix_tables, self.lens, self.starts, self.tables, self.own, scale=self.D**-0.5, out_dtype=F32)
        self.logits = att.view(5, -1) @ self.head
        ops.sample(self.logits, self.u, out=self.next, **self.how)
        self.ids.copy_(self.next)

    def run(self, steps, step):
        out = []
        for i in range(steps):
            self.u.copy_(torch.tensor([s.uniform(i) for s in self.settings]))
            step()
            out.append((self.logits.clone(), self.next.tolist()))
        return out

    def exact(self, tokens):
        """Logits of the last of `tokens` in 64 bits, and how far the step's may be from them."""
        H, K, D = self.H, self.HKV, self.D
        y = self.table[tokens.long()].double() @ self.w.double()
        size = self.table[tokens.long()].double().abs() @ self.w.double().abs()
        n = len(tokens)

        def heads(lo, count, gain):
            x = y[:, lo:lo + count * D].view(n, count, D)
            off = (size[:, lo:lo + count * D].view(n, count, D) * self.WIDTH * 2.0**-24)
            if gain is None:
                return x, off
            r = (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
            off = (off * r + x.abs() * r * ((off * r).amax(-1, keepdim=True) + 72 * 2.0**-24)) * gain.abs()
            x = x * r * gain
            c, s = self.cos[:n, None].double(), self.sin[:n, None].double()
            a, b = x[..., :24], x[..., 24:48]
            oa, ob = off[..., :24], off[..., 24:48]
            both = (oa * c.abs() + ob * s.abs() + 2.0**-22 * (a.abs() + b.abs()), ob * c.abs() + oa * s.abs() + 2.0**-22 * (a.abs() + b.abs()))
            return torch.cat([a * c - b * s, b * c + a * s, x[..., 48:]], -1), torch.cat([*both, off[..., 48:]], -1)

        def stored(x, off, t):
            half, least = {F32: (2.0**-24, 0.0), BF16: (2.0**-8, 0.0), F8: (2.0**-4, 2.0**-10)}[t]
            return x, off + (x.abs() + off) * half + least

        q, qe = (t[-1:] for t in stored(*heads(0, H, self.gains[0].double()), self.query))
        k, ke = stored(*heads(H * D, K, self.gains[1].double()), self.kc.dtype)
        v, ve = stored(*heads((H + K) * D, K, None), self.vc.dtype)
        k, ke, v, ve = (t.repeat_interleave(H // K, 1) for t in (k, ke, v, ve))
        dot = lambda a, b: torch.einsum("hd,nhd->hn", a[0], b) * D**-0.5  # noqa: E731
        s = dot(q, k)
        se = dot(qe, k.abs()) + dot(q.abs() + qe, ke) + dot(q.abs() + qe, k.abs() + ke) * ((D + 2) * 2.0**-24 + 2.0**-17)
        p = torch.softmax(s, 1)
        low, high = p * torch.exp(-2 * se.amax(1, keepdim=True)), p * torch.exp(2 * se.amax(1, keepdim=True))
        o = torch.einsum("hn,nhd->hd", p, v)
        oe = (torch.einsum("hn,nhd->hd", torch.maximum(high - p, p - low), (v - o).abs())
              + torch.einsum("hn,nhd->hd", high, ve) + torch.einsum("hn,nhd->hd", high, v.abs() + ve) * ((n + 8) * 2.0**-24 + 2.0**-17))
        head = self.head.double()
        o, oe = o.reshape(1, -1), oe.reshape(1, -1)
        return (o @ head)[0], (oe @ head.abs() + (o.abs() + oe) @ head.abs() * (H * D * 2.0**-24))[0]


# A weight moves by e^(2 max|ds|) at most (its own exponent and the sum's); as all weights sum to one before and after, only a value's distance from the mean moves the result.
@pytest.mark.parametrize("pool,query", [(F32, F32), (BF16, BF16), (BF16, F32), (F8, BF16)])
def test_steps_against_64_bits(pool, query):
    toy = Toy(pool, query)
    start = toy.ids.tolist()
    done = toy.run(20, toy.step)
    for r in range(5):
        known = torch.cat([toy.prompts[0 if r < 2 else 1], torch.tensor([start[r]], device="cuda")])
        for i, (logits, tokens) in enumerate(done):
            want, far = toy.exact(known)
            off = (logits[r].double() - want).abs()
            assert bool((off <= far).all()), (r, i, (off / far).max().item())
            s = toy.settings[r]
            assert tokens[r] == draw(logits[r].double().cpu().numpy(), s.uniform(i), s), (r, i)
            known = torch.cat([known, torch.tensor([tokens[r]], device="cuda")])


@pytest.mark.parametrize("pool,query", [(BF16, BF16), (F8, BF16), (F32, F32)])
def test_a_graph_of_the_step(pool, query):
    """Captured once, replayed step by step on changing tokens: the eager steps' bits."""
    eager, toy = Toy(pool, query), Toy(pool, query)
    want = eager.run(20, eager.step)
    keep = toy.ids.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        toy.step()
    torch.cuda.current_stream().wait_stream(side)
    toy.ids.copy_(keep)
    toy.own.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        toy.step()
    toy.ids.copy_(keep)
    toy.own.zero_()
    got = toy.run(20, graph.replay)
    assert [t for _, t in got] == [t for _, t in want]
    assert all(torch.equal(a, b) for (a, _), (b, _) in zip(got, want))


# ---------------------------------------------------------------------------------------------- the engine

CONFIG = oracle.model(oracle.layer(), oracle.layer(window=40, ff=0))
SETTINGS = [Sampling(1.0, seed=11), None, Sampling(0.7, 20, 0.9, 0.01, seed=12), Sampling(2.0, 0, 0.95, seed=13), Sampling(0.0)]


def prompt(n):
    return torch.randint(0, 131, (n,), generator=torch.Generator().manual_seed(n)).tolist()


def test_engine_draws_from_the_logits_of_each_step():
    """Requests that wait for pages, each with its own settings: the logits are the plain model's, and every token follows from them."""
    from tlaloc_b200.engine import Engine
    from tlaloc_b200.latent_decoder import LatentDecoder, LatentDecoderConfig

    weights = oracle.make_weights(CONFIG, seed=12)
    model = LatentDecoder(LatentDecoderConfig.from_config(CONFIG), num_blocks=6, max_len=256, dtype=F32, max_tokens=48, max_sequences=4)
    model.load_tensors({k: v.numpy() for k, v in weights.items()})
    seen, sample = [], model.sample

    def recorded(logits, draws):
        seen.append((logits.clone(), draws))
        return sample(logits, draws)

    model.sample = recorded
    prompts = [prompt(n) for n in (3, 70, 20, 1, 130)]
    out = Engine(model).generate(prompts, 12, sampling=SETTINGS)
    want = [oracle.forward(CONFIG, weights, p + o)[len(p) - 1:-1] for p, o in zip(prompts, out)]
    scale = max(float(w.square().mean().sqrt()) for w in want)
    drawn = 0
    for logits, draws in seen:
        for x, (s, i) in zip(logits.double().cpu(), draws):
            if s is None or s.temperature == 0:
                continue
            r = SETTINGS.index(s)
            d = x - want[r][i]
            assert float((d - d.mean()).square().mean().sqrt()) <= 2e-5 * scale  # the error the model's own tests allow in f32
            assert out[r][i] == draw(x.numpy(), s.uniform(i), s)
            drawn += 1
    assert drawn == 36
    assert [out[r] for r in (1, 4)] == [oracle.greedy(CONFIG, weights, prompts[r], 12) for r in (1, 4)]


def test_command_line_draws(tmp_path):
    oracle.save(str(tmp_path), CONFIG, oracle.make_weights(CONFIG, seed=13))
    tokens = ",".join(map(str, prompt(40)))

    def run(*more):
        r = subprocess.run([sys.executable, "-m", "tlaloc_b200", "generate", "--model", str(tmp_path), "--dtype", "float32", "--max-new", "16", "--prompt", tokens, *more],
                           capture_output=True, text=True, cwd=ROOT, timeout=300)
        assert r.returncode == 0, r.stderr
        return [json.loads(line) for line in r.stdout.splitlines()][-1]

    greedy, hot = run(), run("--temperature", "5", "--seed", "3")
    assert run("--temperature", "5", "--top-k", "1") == greedy and hot != greedy and len(hot) == 16
    assert run("--temperature", "5", "--seed", "3") == hot
