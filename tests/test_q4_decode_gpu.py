"""The attention block over the 4-bit cache (kernelfoundry_b200.q4_decode), end to end on the GPU."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


def _reference(block, x, b):
    """The block's output for the last token of sequence b, ``x`` [1, n, hidden], in fp64, the keys and values being what
    the cache holds."""
    import torch

    from kernelfoundry_b200 import kv_read_q4

    n = x.shape[1]
    pos = torch.arange(n, device=x.device)[None]
    q, _, _ = block._project(x, pos)
    slots = block.slots(pos.expand(len(block.lens), n))[b:b + 1].contiguous()
    k, v = kv_read_q4(block.cache, slots, dtype=torch.float16)
    q, k, v = (t.double() for t in (q[0, :, -1], k[0], v[0]))
    G = block.H_q // block.H_kv
    k, v = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
    p = torch.softmax(torch.einsum("hd,hjd->hj", q, k) * block.D ** -0.5, -1)
    o = torch.einsum("hj,hjd->hd", p, v).half().reshape(1, 1, -1)
    return x[:, -1:] + o @ block.w_o


@pytest.mark.parametrize("D,H_q,H_kv,bs", [(128, 8, 2, 16), (64, 6, 3, 32), (256, 4, 1, 64)])
def test_prefill_chunks_then_steps(cuda, D, H_q, H_kv, bs):
    """Two prefill chunks (ragged), three single steps and a two-token draft equal the definition on the cache's values.

    Tolerance: keys and values are rounded to fp16 for the definition (2^-11 relative), the attention output to fp16
    (2^-11), the projection sums hundreds of products: 2^-8 of the output's largest element bounds them together."""
    import torch

    from kernelfoundry_b200.q4_decode import Q4AttentionBlock

    torch.manual_seed(1)
    B, hidden = 3, 256
    block = Q4AttentionBlock(B, 200, hidden, H_q, H_kv, D, bs, device=cuda)
    x = torch.randn(B, 100, hidden, device=cuda).half()
    lens = torch.tensor([40, 1, 17], dtype=torch.int32, device=cuda)
    block.prefill(x[:, :60])
    block.prefill(x[:, 60:], lens, past=60)
    assert block.lens.tolist() == [100, 61, 77]
    seqs = [x[b:b + 1, :60 + int(lens[b])] for b in range(B)]
    for width in (1, 1, 1, 2):
        new = torch.randn(B, width, hidden, device=cuda).half()
        out = block.step(new)
        for b in range(B):
            seqs[b] = torch.cat((seqs[b], new[b:b + 1]), 1)
            want = _reference(block, seqs[b], b)
            err = (out[b, -1] - want[0, 0]).abs().max()
            assert err <= 2.0 ** -8 * want.abs().max(), (width, b, err)
    assert block.lens.tolist() == [105, 66, 82]


def test_step_from_a_captured_graph(cuda):
    """Replays advance the lengths on the device and give what eager steps give."""
    import torch

    from kernelfoundry_b200.q4_decode import Q4AttentionBlock

    outs = []
    for graphed in (False, True):
        torch.manual_seed(2)
        block = Q4AttentionBlock(2, 64, 256, 8, 2, 128, device=cuda)
        x = torch.randn(2, 20, 256, device=cuda).half()
        block.prefill(x, torch.tensor([20, 7], dtype=torch.int32, device=cuda))
        token = torch.randn(2, 1, 256, device=cuda).half()
        block.step(token)
        if not graphed:
            outs.append([block.step(token).clone() for _ in range(4)])
            continue
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block.step(token)
        got = []
        for _ in range(4):
            graph.replay()
            got.append(out.clone())
        outs.append(got)
        assert block.lens.tolist() == [25, 12]
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D,H_q,H_kv,widths", [(128, 8, 2, (1, 2, 5, 16)), (64, 6, 3, (1, 32)), (256, 4, 1, (1, 16))])
def test_steps_use_the_blocks_own_workspace(cuda, monkeypatch, D, H_q, H_kv, widths):
    """Eager or captured, for steps of any width: no call makes a workspace (which a graph would fill again at each replay)."""
    import torch

    from kernelfoundry_b200 import kv_cache
    from kernelfoundry_b200.q4_decode import Q4AttentionBlock

    def none(*_):
        raise AssertionError("the stream's workspace was asked for")

    monkeypatch.setattr(kv_cache, "_workspace", none)
    torch.manual_seed(3)
    block = Q4AttentionBlock(2, 200, 256, H_q, H_kv, D, device=cuda)
    block.prefill(torch.randn(2, 20, 256, device=cuda).half())
    for w in widths:
        x = torch.randn(2, w, 256, device=cuda).half()
        block.step(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block.step(x)
        block.lens -= w                                  # the same step twice: eager, then replayed
        want = block.step(x).clone()
        block.lens -= w
        graph.replay()
        assert torch.equal(out, want)
