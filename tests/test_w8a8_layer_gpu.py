"""A decoder layer of an 8-bit checkpoint out of the operators, as a serving loop runs it: norm and q/k/v product, rotation and append, attention over
the cache, output product, feed-forward behind its norm; a prompt, then a draft tree's rows, then single tokens."""
import pytest
import torch

import w8a8_cases as ref
from test_rotary_gpu import definition

pytestmark = pytest.mark.gpu
BF16, I32 = torch.bfloat16, torch.int32
HIDDEN, HEADS, KV, DIM, INTER, BUDGET = 1024, 8, 2, 128, 1536, 512


def attention(q, k, v, scale):
    """q [t, heads, d] over the cache rows [n, kv, d], the last t of them its own: 64 bits"""
    t, n = q.shape[0], k.shape[0]
    k, v = (a.double().repeat_interleave(HEADS // KV, 1) for a in (k, v))
    s = torch.einsum("thd,nhd->htn", q.double(), k) * scale
    s = s.masked_fill(torch.arange(n, device="cuda")[None] > torch.arange(n - t, n, device="cuda")[:, None], float("-inf"))
    return torch.einsum("htn,nhd->thd", torch.softmax(s, -1), v).reshape(t, -1)


def test_layer():
    import cpmcu.C as C
    from cpmcu import rotary, w8a8
    g = torch.Generator("cuda").manual_seed(0)

    def weight(out, width):
        w = (torch.randn(out, width, generator=g, device="cuda") / width ** 0.5).to(BF16)
        q, s = w8a8.quantize(w)
        return (q, s), w8a8.PackedLinear(q, s)
    qkv_w, qkv_p = weight((HEADS + 2 * KV) * DIM, HIDDEN)
    o_w, o_p = weight(HIDDEN, HEADS * DIM)
    gate, up = weight(INTER, HIDDEN)[0], weight(INTER, HIDDEN)[0]
    down_w, down_p = weight(HIDDEN, INTER)
    gate_up = w8a8.PackedGateUp(*gate, *up)
    n1, n2 = (1 + 0.1 * torch.randn(2, HIDDEN, generator=g, device="cuda")).to(BF16)
    inv, factor = rotary.frequencies(DIM, 10000.0, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 128})
    inv = inv.cuda()
    k_cache, v_cache = torch.zeros(2, BUDGET, KV * DIM, dtype=BF16, device="cuda")
    length, scale = 0, DIM ** -0.5
    tokens = torch.randn(400, HIDDEN, generator=g, device="cuda").to(BF16)
    residual = torch.randn(400, HIDDEN, generator=g, device="cuda").to(BF16)     # what the layer before adds
    for rows in (300, 60, 1, 1, 7):
        x, d = tokens[length:length + rows].contiguous(), residual[length:length + rows].contiguous()
        pos = torch.arange(length, length + rows, dtype=I32, device="cuda")
        kv_len = torch.tensor([length + rows], dtype=I32, device="cuda")

        # the layer, call after call
        qkv, h = w8a8.linear(x, qkv_p, norm_weight=n1, delta=d)
        q = rotary.append(qkv, HEADS, KV, DIM, inv, pos, k_cache, v_cache, pos, factor=factor)
        a = torch.empty(rows, HEADS * DIM, dtype=BF16, device="cuda")
        C.call("cpmcu_tree_attention", q.data_ptr(), HEADS * DIM, k_cache.data_ptr(), v_cache.data_ptr(), BUDGET, rows, HEADS, KV, kv_len.data_ptr(), 0, None,
               None, 0, 0, 1, a.data_ptr(), HEADS * DIM)
        o = w8a8.linear(a, o_p)
        y, h2 = w8a8.gated_ffn(h, gate_up, down_p, norm_weight=n2, delta=o)

        # each call on its actual inputs, in 64 bits
        t = ref.residual(x, d, 1.0)
        assert float((h.double() - t.double()).abs().max()) <= float(t.double().abs().max()) * 2.0 ** -7
        want, tol, _ = ref.linear(h, *qkv_w, norm_weight=n1)
        assert bool(((qkv.double() - want).abs() <= tol).all())
        want, values, tol = definition(qkv, HEADS, KV, DIM, inv, pos, DIM, False, factor)
        assert bool(((q.double().unflatten(1, (HEADS, DIM)) - want[:, :HEADS]).abs() <= tol[:, :HEADS]).all())
        assert bool(((k_cache[length:length + rows].double().unflatten(1, (KV, DIM)) - want[:, HEADS:]).abs() <= tol[:, HEADS:]).all())
        assert torch.equal(v_cache[length:length + rows].double().unflatten(1, (KV, DIM)), values)
        length += rows
        want = attention(q.view(rows, HEADS, DIM), k_cache[:length].view(length, KV, DIM), v_cache[:length].view(length, KV, DIM), scale)
        # bf16 probabilities and values: the tolerance of the attention's own tests
        assert float((a.double() - want).abs().max()) < 0.03
        want, tol, _ = ref.linear(a, *o_w)
        assert bool(((o.double() - want).abs() <= tol).all())
        want, tol, _ = ref.ffn(h2, *gate, *up, *down_w, norm_weight=n2)
        assert bool(((y.double() - want).abs() <= tol).all())
        C.stream_check(torch.cuda.current_stream().cuda_stream)
    assert not bool(k_cache[length:].any()) and not bool(v_cache[length:].any())
