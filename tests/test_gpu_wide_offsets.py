"""Operands whose element offsets pass 2^31: a cache with a huge row stride, a table and logits of more than 2^31 elements.
Each result equals, bit for bit, that of the same values in compact memory (addresses decide no order of a sum; alignment
is the same)."""
import pytest
import torch

gpu = pytest.mark.gpu


@gpu
def test_attention_over_far_rows(dev):
    from deeprec_amd import kernels as K
    L, D, step = 9, 64, 2 ** 28
    buf = torch.empty(8 * step + 4 * D, dtype=torch.bfloat16, device=dev)
    far = [buf.as_strided((1, L, 1, D), (0, step, D, 1), i * D) for i in range(3)]
    g = torch.Generator().manual_seed(1)
    near = [torch.randn((1, L, 1, D), generator=g).to(torch.bfloat16).to(dev) for _ in range(3)]
    for a, b in zip(far, near):
        a.copy_(b)
    go = torch.randn((1, L, 1, D), generator=g).to(torch.bfloat16).to(dev)
    a, b = (K.window_attn_forward(*t, window=4, sinks=1) for t in (far, near))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for x, y in zip(K.window_attn_backward(*far, *a, go, window=4, sinks=1), K.window_attn_backward(*near, *b, go, window=4, sinks=1)):
        assert torch.equal(x, y)
    assert torch.equal(K.window_attn_token(far[0][:, -1], *far[1:], window=4, sinks=1),
                       K.window_attn_token(near[0][:, -1], *near[1:], window=4, sinks=1))


@gpu
def test_embedding_of_a_large_table(dev):
    from deeprec_amd import kernels as K
    rows, d = 2 ** 24 + 5, 128                                               # 2^31 + 640 elements
    table = torch.empty((rows, d), dtype=torch.bfloat16, device=dev)
    ids = torch.tensor([0, rows - 1, 5, 2 ** 24, rows - 1, rows], device=dev)
    for i in (0, 5, 2 ** 24, rows - 1):
        table[i] = torch.randn(d, device=dev).to(torch.bfloat16)
    out = K.embed_forward(table, ids, scale=2.0)
    assert torch.equal(out[:5], table[ids[:5]] * 2) and not bool(out[5].any())
    del table
    grad = K.embed_backward(out, ids, rows)
    assert torch.equal(grad[rows - 1], (out[1].float() + out[4].float()).to(torch.bfloat16))
    assert torch.equal(grad[2 ** 24], out[3]) and torch.equal(grad[0], out[0])
    assert int((grad.view(torch.int16) != 0).any(1).sum()) == 4


@gpu
def test_logprobs_of_far_rows(dev):
    from deeprec_amd import kernels as K
    V, ld = 3001, 2 ** 31 + 8
    buf = torch.empty(ld + V, dtype=torch.float16, device=dev)
    near = torch.randn((2, V), device=dev).half()
    far = buf.as_strided((2, V), (ld, 1))
    far.copy_(near)
    pad = torch.empty((2, V + 7), dtype=torch.float16, device=dev)           # rows 16 bytes apart from the grid alike: 3008 = 8 x 376
    pad[:, :V] = near
    t = torch.tensor([7, 3000], device=dev)
    a, b = K.item_logprobs_forward(far, t, K=5), K.item_logprobs_forward(pad[:, :V], t, K=5)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    g = torch.ones(2, device=dev)
    assert torch.equal(K.item_logprobs_backward(far, t, a.lse, a.entropy, g), K.item_logprobs_backward(pad[:, :V], t, b.lse, b.entropy, g))
