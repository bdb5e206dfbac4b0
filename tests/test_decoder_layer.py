"""The decoder-layer operators together, as a model runs them: per-token
quantisation, QKV product, cache append, attention over the cache, output
product with the residual - a ragged prompt, then single tokens, eager and
from a captured graph - against a plain 64-bit implementation."""
import numpy as np
import pytest
import torch

from iconnx_b200 import ops
from iconnx_b200.kv_cache import KvCache, gpu_kv_cache_append, gpu_kv_cache_attention
from tests import decoder_reference as ref

DEV = "cuda:0"
WIDTH, HEADS, KV, DIM = 256, 4, 2, 64


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def f64(t):
    return t.detach().cpu().double().numpy()


class Layer:
    def __init__(self, dtype, bits, seed):
        g = torch.Generator().manual_seed(seed)
        self.dtype = dtype
        n = (HEADS + 2 * KV) * DIM
        self.w = [torch.randint(-127, 128, s, generator=g, dtype=torch.int8) for s in ((WIDTH, n), (HEADS * DIM, WIDTH))]
        self.ws = [(0.5 + torch.rand(s, generator=g)) / (73 * 16) for s in (n, WIDTH)]
        self.bias = torch.randn(n, generator=g) * 0.1
        self.pw = [ops.prepare_weight(w.to(DEV)) for w in self.w]
        self.cw = [s.to(DEV) for s in self.ws]
        self.cb = self.bias.to(DEV)
        self.cache = KvCache(24, 16, KV, DIM, bits, 32, DEV)

    def __call__(self, x, table, lens, cu=None):
        q, s = ops.gpu_quantize_per_token(x)
        qkv = ops.gpu_matmul_integer_scaled(q, s, self.pw[0], self.cw[0], bias=self.cb, out_dtype=self.dtype)
        qkv = qkv.view(len(x), HEADS + 2 * KV, DIM)
        gpu_kv_cache_append(self.cache, qkv[:, HEADS:HEADS + KV], qkv[:, HEADS + KV:], table, lens, cu)
        a = gpu_kv_cache_attention(self.cache, qkv[:, :HEADS], table, lens, cu)
        q, s = ops.gpu_quantize_per_token(a.view(len(x), -1))
        return qkv, a, ops.gpu_matmul_integer_scaled(q, s, self.pw[1], self.cw[1], residual=x, out_dtype=self.dtype)


class Plain:
    """Fed stage by stage with what the layer computed, so that each stage's own
    error is what is bounded: a code on the other side of a half would change
    what follows by a whole step."""

    def __init__(self, layer, bits, batch):
        self.l, self.bits = layer, bits
        self.k, self.v = ([np.zeros((0, KV, DIM)) for _ in range(batch)] for _ in range(2))

    def check(self, x, qkv, a, out, news):
        l, dt = self.l, self.l.dtype
        q, s = ref.quantize_per_token(f64(x))
        acc, want = ref.scaled_product(q, s, l.w[0].numpy(), l.ws[0].numpy(), l.bias.numpy())
        got = f64(qkv).reshape(want.shape)
        tol = ref.rounding(want, 5 * 2.0 ** -24 * (np.abs(want) + 2 * np.abs(l.bias.numpy())), dt)
        assert (np.abs(got - want) <= tol).all()
        at = 0
        for b, n in enumerate(news):
            rows = f64(qkv[at:at + n])
            self.k[b] = np.concatenate([self.k[b], ref.cached_values(rows[:, HEADS:HEADS + KV], self.bits, 32)])
            self.v[b] = np.concatenate([self.v[b], ref.cached_values(rows[:, HEADS + KV:], self.bits, 32)])
            want = ref.attention(rows[:, :HEADS], self.k[b], self.v[b], DIM ** -0.5)
            tol = ref.attention_tolerance(rows[:, :HEADS], self.k[b], self.v[b], DIM ** -0.5, dt, want)
            assert (np.abs(f64(a[at:at + n]) - want) <= tol).all()
            at += n
        q, s = ref.quantize_per_token(f64(a).reshape(at, -1))
        acc, want = ref.scaled_product(q, s, l.w[1].numpy(), l.ws[1].numpy(), residual=f64(x))
        tol = ref.rounding(want, 5 * 2.0 ** -24 * (np.abs(want) + 2 * np.abs(f64(x))), dt)
        assert (np.abs(f64(out) - want) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [4, 8])
def test_prompt_then_decode(dtype, bits):
    layer = Layer(dtype, bits, 1)
    lens = [37, 1, 80]
    plain = Plain(layer, bits, len(lens))
    table = i32(np.random.RandomState(0).permutation(24).reshape(3, 8))
    g = torch.Generator(DEV).manual_seed(2)

    def tokens(n):
        return torch.randn(n, WIDTH, generator=g, device=DEV).to(dtype)

    x = tokens(sum(lens))
    plain.check(x, *layer(x, table, i32(lens), i32([0, *np.cumsum(lens)])), lens)
    for step in range(3):
        lens = [n + 1 for n in lens]
        x = tokens(3)
        plain.check(x, *layer(x, table, i32(lens)), [1, 1, 1])
    # the same step captured, replayed with other tokens and lengths
    buf, dev_lens = tokens(3), i32(lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = layer(buf, table, dev_lens)
    for step in range(3):
        lens = [n + 1 for n in lens]
        x = tokens(3)
        buf.copy_(x)
        dev_lens.copy_(i32(lens))
        graph.replay()
        torch.cuda.synchronize()
        plain.check(x, *outs, [1, 1, 1])
