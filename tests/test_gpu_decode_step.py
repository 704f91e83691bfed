"""GPU: the few-bit entry points together, as a token-by-token transformer uses them.

One pre-norm layer: norm + int8 rows -> 4-bit q, k, v -> cache append -> attention -> 4-bit output
projection -> residual + norm -> 4-bit FFN with GELU -> residual + norm -> an int8 head (sdq_qgemm's
second half).  A prompt chunk first, then single tokens from a captured graph whose tables move on.
Every stage is checked from the inputs it really had, so the stages' own bounds apply.
"""
import ctypes as C

import numpy as np
import pytest
import torch

from fewbit_util import DT, Pool, attention64, attention_tolerance, int8_rows, ptr
from test_gpu_rmsnorm import restate
from test_gpu_w4 import full_range, reference, tolerance, upload
from util import packed_weights

pytestmark = pytest.mark.gpu

D, HEADS, KV, HD, FFN, GROUP, VOCAB = 256, 8, 2, 64, 640, 64, 384


class Layer:
    def __init__(self, sdq, rng, name):
        self.sdq, self.name, self.code = sdq, name, DT[name][0]
        shapes = {"q": (HEADS * HD, D), "k": (KV * HD, D), "v": (KV * HD, D), "o": (D, HEADS * HD), "up": (FFN, D), "down": (D, FFN)}
        self.host = {n: full_range(rng, N, K, GROUP, "bf16") for n, (N, K) in shapes.items()}
        self.w = {n: upload(sdq, q, sc, GROUP, "bf16") for n, (q, sc) in self.host.items()}
        self.bias = torch.from_numpy(rng.standard_normal(FFN).astype(np.float32)).cuda()
        self.norms = [torch.from_numpy((1 + 0.2 * rng.standard_normal(D)).astype(np.float32)).cuda() for _ in range(3)]

    def buffers(self, M):
        dt, e = DT[self.name][1], lambda *s, t=None: torch.zeros(*s, device="cuda", dtype=t or DT[self.name][1])
        b = {"x": e(M, D), "sum1": e(M, D), "sum2": e(M, D), "q": e(M, HEADS, HD), "k": e(M, KV, HD), "v": e(M, KV, HD),
             "att": e(M, HEADS, HD), "o": e(M, D), "up": e(M, FFN), "down": e(M, D), "logits": torch.zeros(M, VOCAB, device="cuda")}
        for i in range(3):
            b["a%d" % i], b["s%d" % i] = e(M, D, t=torch.int8), e(M, t=torch.float32)
        return b

    def step(self, b, M, pool, head, stream=None):
        f, t = self.sdq, self.code

        def linear(n, src, dst, bias=None, gelu=False, rows=None):
            if rows is None:
                f.w4_matmul(self.w[n], ptr(src), t, M, ptr(dst), t, bias_ptr=ptr(bias), gelu=gelu, stream=stream)
            else:
                f.w4_matmul(self.w[n], ptr(src), 3, M, ptr(dst), t, a_scale_ptr=ptr(rows), bias_ptr=ptr(bias), gelu=gelu, stream=stream)

        f.rmsnorm_quantize(ptr(b["x"]), t, M, D, ptr(b["a0"]), ptr(b["s0"]), weight_ptr=ptr(self.norms[0]), stream=stream)
        for n in ("q", "k", "v"):
            linear(n, b["a0"], b[n], rows=b["s0"])
        f.kv_append(pool.cache, pool.seqs, ptr(b["k"]), ptr(b["v"]), t, M, stream=stream)
        f.kv_attention(pool.cache, pool.seqs, ptr(b["q"]), t, M, HEADS, ptr(b["att"]), causal=True, stream=stream)
        linear("o", b["att"], b["o"])
        f.rmsnorm_quantize(ptr(b["o"]), t, M, D, ptr(b["a1"]), ptr(b["s1"]), weight_ptr=ptr(self.norms[1]), residual_ptr=ptr(b["x"]),
                           sum_ptr=ptr(b["sum1"]), stream=stream)
        linear("up", b["a1"], b["up"], self.bias, True, rows=b["s1"])
        linear("down", b["up"], b["down"])
        f.rmsnorm_quantize(ptr(b["down"]), t, M, D, ptr(b["a2"]), ptr(b["s2"]), weight_ptr=ptr(self.norms[2]),
                           residual_ptr=ptr(b["sum1"]), sum_ptr=ptr(b["sum2"]), stream=stream)
        f._ck(f.lib.sdq_qgemm_prequantized(head, ptr(b["a2"]), ptr(b["s2"]), M, ptr(b["logits"]), None, None, 0, stream))

    def check(self, b, M, pool, oracle, head_np):
        name = self.name
        c = {n: t.detach().cpu() for n, t in b.items()}
        w = [n.cpu() for n in self.norms]

        def norm(i, x, res, total):
            s, _, aq, sc = restate(x, res, w[i], 1e-6, name)
            assert np.array_equal(c["a%d" % i].numpy(), aq) and np.array_equal(c["s%d" % i].numpy(), sc)
            assert total is None or torch.equal(total, s)

        def linear(n, x, xs, got, bias=None, gelu=False):
            q, sc = self.host[n]
            want, mag = reference(x.reshape(M, -1).double().numpy(), xs, q, sc, GROUP, bias, gelu)
            tol = tolerance(want, mag, q.shape[1], GROUP, name, gelu)
            assert (np.abs(got.reshape(M, -1).double().numpy() - want) <= tol).all(), n

        norm(0, c["x"], None, None)
        for n in ("q", "k", "v"):
            linear(n, c["a0"], c["s0"].numpy(), c[n])
        for i in range(len(pool.keys)):
            n, first = pool.new[i], int(pool.starts[i])
            for which in ("k", "v"):
                codes, sc = int8_rows(c[which][first:first + n].float().numpy())
                stored = pool.dense(i, which)[pool.keys[i] - n:]
                assert np.array_equal(stored, codes.astype(np.float64) * sc[..., None].astype(np.float64))
            want, *sizes = attention64(pool, c["q"].double().numpy(), HEADS, HD ** -0.5, True, i)
            tol = attention_tolerance(name, pool, i, HEADS, want, *sizes)
            assert (np.abs(c["att"][first:first + n].double().numpy() - want) <= tol).all()
        linear("o", c["att"], None, c["o"])
        norm(1, c["o"], c["x"], c["sum1"])
        linear("up", c["a1"], c["s1"].numpy(), c["up"], self.bias.cpu().numpy(), True)
        linear("down", c["up"], None, c["down"])
        norm(2, c["down"], c["sum1"], c["sum2"])
        acc = oracle.dot_s32(c["a2"].numpy(), head_np[0])
        assert np.array_equal(c["logits"].numpy(), oracle.rescale(acc, c["s2"].numpy(), head_np[1]))


@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_prompt_then_tokens(sdq, oracle, name):
    rng = np.random.default_rng(77)
    layer = Layer(sdq, rng, name)
    head_np = packed_weights(rng, VOCAB, D, oracle)
    head = sdq.weight_upload(*head_np)
    prompt, tokens = [37, 5, 90], 4
    pool = Pool(sdq, rng, prompt, [p + tokens for p in prompt], KV, 16, HD)      # room for the tokens to come
    pool.keys = list(prompt)
    pool.refresh()
    M = sum(prompt)
    b = layer.buffers(M)
    b["x"].copy_(torch.from_numpy(rng.standard_normal((M, D)).astype(np.float32)))
    layer.step(b, M, pool, head)
    torch.cuda.synchronize()
    layer.check(b, M, pool, oracle, head_np)
    # single tokens: the same tables object, now one row a sequence, from a captured graph
    B = len(prompt)
    pool.new, pool.starts, pool.rows = [1] * B, np.arange(B + 1, dtype=np.int32), B
    pool.keys = [p + 1 for p in prompt]
    pool.refresh()
    b = layer.buffers(B)
    st, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    sp = C.c_void_p(st.cuda_stream)
    with torch.cuda.stream(st):
        layer.step(b, B, pool, head, sp)              # sizes the int8 GEMM's scratch of this stream
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=st):
            layer.step(b, B, pool, head, sp)
    for i in range(tokens):
        pool.keys = [p + 1 + i for p in prompt]
        pool.d_len.copy_(torch.tensor(pool.keys, dtype=torch.int32))
        b["x"].copy_(torch.from_numpy(rng.standard_normal((B, D)).astype(np.float32)))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        layer.check(b, B, pool, oracle, head_np)
    for h in list(layer.w.values()) + [head]:
        sdq.weight_release(h)
