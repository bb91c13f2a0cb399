"""The student decoder's operators against their definitions in 64 bits, at the sizes and masks where they can go wrong."""
import math

import pytest
import torch

import student_oracle as oracle

pytestmark = pytest.mark.gpu
bf = torch.bfloat16


def _rand(g, *shape, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(bf)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- norms of queries and keys, rotation ------------------------------------------------------------------------
@pytest.mark.parametrize("B, S, heads, kv, D, weights", [
    (1, 1, 1, 1, 8, bf), (1, 1, 4, 2, 64, torch.float32), (2, 3, 4, 2, 64, bf), (1, 37, 32, 8, 128, bf), (3, 5, 6, 3, 96, torch.float32), (1, 9, 2, 1, 256, bf),
    (2, 11, 3, 1, 24, bf), (1, 300, 7, 7, 40, torch.float32), (2, 700, 8, 2, 128, torch.float32), (1, 33, 5, 1, 136, bf),
])
def test_qk_norm_rope(B, S, heads, kv, D, weights):
    from rocm_systems_b200.ops import attention, train_ops

    g = _gen(B * 1000 + S)
    qkv = _rand(g, B, S, heads + 2 * kv, D).requires_grad_(True)
    wq, wk = ((1 + 0.3 * torch.randn(D, device="cuda", generator=g)).to(weights).requires_grad_(True) for _ in range(2))
    table = train_ops.rope_table(S + 3, D, 10000.0, "cuda")
    grads = tuple(_rand(g, B, S, n, D).transpose(1, 2) for n in (heads, kv, kv))
    out = attention.qk_norm_rope(qkv, wq, wk, table, heads, kv, 1e-5)
    back = torch.autograd.grad(out, (qkv, wq, wk), grads)
    ref = oracle.qk_norm_rope(qkv, wq, wk, table, heads, kv, 1e-5, grads)
    for n, t in zip(("q", "k", "v", "dqkv", "dwq", "dwk"), (*out, *back)):
        oracle.off(n, t, ref)
    assert back[1].dtype == weights and out[2].data_ptr() == qkv.data_ptr() + 2 * (heads + kv) * D


def test_qk_norm_rope_with_other_layouts():
    """Gradients that are no [B, S, heads, D] memory, broadcast or off 16 bytes; a packed projection that is a slice of something wider."""
    from rocm_systems_b200.ops import attention, train_ops

    B, S, heads, kv, D = 2, 13, 4, 2, 64
    g = _gen(5)
    wide = _rand(g, B, S, heads + 2 * kv, D + 4)
    qkv = wide[..., 4:].detach().requires_grad_(True)
    wq, wk = (torch.ones(D, device="cuda", requires_grad=True) for _ in range(2))
    table = train_ops.rope_table(S, D, 10000.0, "cuda")
    out = attention.qk_norm_rope(qkv, wq, wk, table, heads, kv, 1e-5)
    dq = _rand(g, B, heads, S, D)                                # heads outside positions
    dk = _rand(g, 1, 1, 1, D).expand(B, kv, S, D)                # one gradient for all
    dv = _rand(g, B * kv * S * D + 1)[1:].view(B, kv, S, D)      # 2 bytes off
    back = torch.autograd.grad(out, (qkv, wq, wk), (dq, dk, dv))
    ref = oracle.qk_norm_rope(qkv, wq, wk, table, heads, kv, 1e-5, (dq, dk, dv))
    for n, t in zip(("q", "k", "v", "dqkv", "dwq", "dwk"), (*out, *back)):
        oracle.off(n, t, ref)
    (only_v,) = torch.autograd.grad(attention.qk_norm_rope(qkv, wq, wk, table, heads, kv)[2], qkv, dv)   # no gradient for q and k
    assert torch.equal(only_v[:, :, heads + kv:], dv.transpose(1, 2)) and not only_v[:, :, :heads + kv].any()


def test_qk_norm_rope_rows_of_zeros_and_one_bad_row():
    """A row of zeros answers zeros (eps keeps the norm finite); an infinite value stays in its own head's row."""
    from rocm_systems_b200.ops import attention, train_ops

    qkv = _rand(_gen(1), 1, 6, 4, 64)
    qkv[0, 2, 1] = 0
    qkv[0, 4, 0, 7] = math.inf
    w = torch.ones(64, device="cuda")
    q, k, v = attention.qk_norm_rope(qkv, w, w, train_ops.rope_table(6, 64, 10000.0, "cuda"), 2, 1)
    assert not q[0, 1, 2].any()
    bad = ~torch.isfinite(q).all(-1)
    assert bool(bad[0, 0, 4]) and int(bad.sum()) == 1 and bool(torch.isfinite(k).all())


# ---- attention with a window and sinks ---------------------------------------------------------------------------
def _attention_inputs(seed, B, H, KV, S, D):
    g = _gen(seed)
    packed = _rand(g, B, S, H + 2 * KV, D)
    q, k, v = (packed[:, :, a:b].transpose(1, 2).detach().requires_grad_(True) for a, b in ((0, H), (H, H + KV), (H + KV, H + 2 * KV)))
    return q, k, v, _rand(g, B, S, H, D).transpose(1, 2)


def _check_attention(q, k, v, dout, window, sinks, lengths=None, scale=None):
    from rocm_systems_b200.ops import attention

    out = attention.window_attention(q, k, v, window, sinks, lengths, scale)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), dout)), out=out)
    ref = oracle.attention(q, k, v, window, sinks, lengths, 1 / math.sqrt(q.shape[-1]) if scale is None else scale, dout)
    for n in ("out", "dq", "dk", "dv"):
        oracle.off(n, got[n], ref)
    return got


@pytest.mark.parametrize("S", [1, 2, 7, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 384, 517])
@pytest.mark.parametrize("window, sinks", [(0, 0), (1, 0), (50, 3), (128, 0), (130, 140), (300, 1)])
def test_window_attention_lengths_and_windows(S, window, sinks):
    _check_attention(*_attention_inputs(S, 1, 4, 2, S, 64), window, sinks)


@pytest.mark.parametrize("B, H, KV, S, D", [(1, 1, 1, 5, 8), (2, 3, 1, 150, 128), (1, 4, 4, 300, 128), (2, 6, 2, 129, 96), (1, 8, 1, 260, 40), (3, 2, 2, 70, 16), (1, 5, 5, 140, 72)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (70, 5)])
def test_window_attention_heads(B, H, KV, S, D, window, sinks):
    _check_attention(*_attention_inputs(S + D, B, H, KV, S, D), window, sinks)


@pytest.mark.parametrize("B, S, window, sinks", [(24, 1400, 100, 200), (64, 600, 40, 300), (2, 700, 1, 700)])
def test_window_attention_many_sinks(B, S, window, sinks):
    """As many key tiles with sinks as need no splitting of their later queries, or little of it."""
    _check_attention(*_attention_inputs(B, B, 8, 8, S, 64), window, sinks)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window, sinks", [(300, 4), (0, 0), (513, 129)])
def test_window_attention_many_tiles(D, window, sinks):
    _check_attention(*_attention_inputs(3, 1, 4, 2, 1700, D), window, sinks)


@pytest.mark.parametrize("lengths", [(0, 1, 200), (200, 200, 200), (129, 128, 127), (-5, 64, 1000)])
@pytest.mark.parametrize("D, window, sinks", [(64, 0, 0), (128, 40, 2), (128, 1, 0)])
def test_window_attention_padded_batches(lengths, D, window, sinks):
    """What lies behind a sequence's end (here NaN and infinities) is not used; its rows answer zeros and get zero gradients."""
    q, k, v, dout = _attention_inputs(11, 3, 4, 2, 200, D)
    L = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for t in (q, k, v, dout):
        for b, n in enumerate(lengths):
            n = min(max(n, 0), 200)
            t.data[b, :, n:] = math.nan
            t.data[b, :, n:, ::3] = math.inf
    got = _check_attention(q, k, v, dout, window, sinks, L)
    for n, t in got.items():
        for b, m in enumerate(lengths):
            assert not t[b, :, min(max(m, 0), 200):].any(), n


def test_window_attention_large_scores():
    """Scores far apart: nearly one-hot rows, a maximum that moves at every tile, and a given scale."""
    q, k, v, dout = _attention_inputs(2, 1, 2, 1, 400, 64)
    k.data *= torch.linspace(0.1, 8, 400, device="cuda").to(bf).view(1, 1, 400, 1)
    _check_attention(q, k, v, dout, 0, 0)
    _check_attention(q, k, v, dout, 150, 3, scale=0.5)
    _check_attention(q, k, v, dout, 150, 3, scale=0.0)


@pytest.mark.parametrize("S, window, sinks", [(2, 0, 0), (3, 1, 2), (5, 0, 0), (40, 2, 0), (700, 2, 1), (700, 100, 28), (700, 100, 29), (700, 60, 4), (700, 60, 5), (1100, 1, 1),
                                              (256, 0, 0), (256, 9, 3), (257, 0, 0)])
def test_window_attention_rows_that_see_few_keys(S, window, sinks):
    """Peaked rows of a few keys, where a gradient is a small difference of weights (the tolerance knows how the weights are rounded)."""
    q, k, v, dout = _attention_inputs(S + window, 2, 4, 2, S, 64)
    q.data *= 2
    _check_attention(q, k, v, dout, window, sinks)


def test_window_attention_strides():
    """Layouts other than the packed projection's: heads outside positions, rows off 16 bytes, one key head's memory for all, a transposed gradient."""
    B, H, KV, S, D = 2, 4, 2, 150, 64
    g = _gen(9)
    q = _rand(g, B, H, S, D).requires_grad_(True)
    k = _rand(g, B * KV * S * D + 1)[1:].view(B, KV, S, D).detach().requires_grad_(True)
    v = _rand(g, B, 1, S, D).expand(B, KV, S, D).detach().requires_grad_(True)
    dout = _rand(g, B, H, D, S).transpose(2, 3)
    _check_attention(q, k, v, dout, 33, 2)
    q = _rand(g, B, S, H, D + 8)[..., :D].transpose(1, 2).detach().requires_grad_(True)
    _check_attention(q, k, v, _rand(g, 1, 1, 1, 1).expand(B, H, S, D), 0, 0)


def test_window_attention_repeats_bit_by_bit_and_in_graphs():
    """Two runs, a run on another stream and a replayed graph give the same bits; two captured graphs keep their results apart."""
    from rocm_systems_b200.ops import attention

    q, k, v, dout = _attention_inputs(4, 2, 4, 2, 700, 128)

    def step():  # detached: an eager graph of the same leaves that is still alive forbids capturing a backward pass
        out = attention.window_attention(q, k, v, 200, 5)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), dout))

    first = step()
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    del again
    graphs, kept = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            kept.append(step())
    for gr in (*graphs, *graphs):
        gr.replay()
    torch.cuda.synchronize()
    for res in kept:
        assert all(torch.equal(a, b) for a, b in zip(first, res))
    with torch.no_grad():
        assert torch.equal(attention.window_attention(q, k, v, 200, 5), first[0])


# ---- distillation ------------------------------------------------------------------------------------------------
def _distill_inputs(seed, T, V, K, ids=torch.int64, values=torch.float32):
    g = _gen(seed)
    logits = _rand(g, T, V, scale=2.5)
    i = torch.stack([torch.randperm(V, device="cuda", generator=g)[:K] for _ in range(T)])
    y = torch.randn(T, K, device="cuda", generator=g) * 2
    tgt = torch.where(torch.rand(T, device="cuda", generator=g) < 0.5, i[:, 0], torch.randint(0, V, (T,), device="cuda", generator=g))
    if T > 2:
        tgt[1], tgt[2] = -100, V
    return logits, tgt, i.to(ids), y.to(values)


def _check_distill(logits, tgt, ids, values, weight, tau, scale, grad=None):
    from rocm_systems_b200.ops import train_ops

    ref = oracle.distill(logits, tgt, ids, values, weight, tau, scale)
    before = logits.clone()
    loss, out = train_ops.distill_loss(logits, tgt, ids, values, weight, tau, scale, grad=grad)
    oracle.off("loss", loss, ref)
    oracle.off("grad", out, ref)
    assert grad is None or out is grad
    if grad is not logits:
        assert torch.equal(logits, before)
    return loss, out


@pytest.mark.parametrize("T, V, K", [(1, 1, 1), (1, 8, 3), (5, 7, 7), (3, 1000, 16), (9, 1003, 5), (4, 4096, 1), (6, 32000, 64), (4, 50257, 33), (5, 128256, 64), (2, 300000, 200),
                                     (3, 5000, 1024), (3, 32768, 9), (3, 32776, 9), (2, 65600, 9), (1, 262145, 5), (1, 851968, 5)])
@pytest.mark.parametrize("weight, tau", [(0.5, 2.0), (1.0, 1.0), (0.0, 3.0), (0.3, 3.0), (0.6, 4.0), (0.4, 1.0), (1.0, 2.5), (0.7, 2.5)])
def test_distill_loss(T, V, K, weight, tau):
    _check_distill(*_distill_inputs(T + V, T, V, K), weight, tau, 1 / T)


@pytest.mark.parametrize("weight, tau", [(0.5, 0.01), (1.0, 0.01), (0.5, 0.1), (0.5, 30.0), (0.5, 100.0), (1.0, 100.0)])
def test_distill_loss_temperature_range(weight, tau):
    _check_distill(*_distill_inputs(11, 4, 33000, 20), weight, tau, 0.25)


@pytest.mark.parametrize("ids, values", [(torch.int32, torch.float32), (torch.int32, bf), (torch.int64, bf)])
def test_distill_loss_types(ids, values):
    _check_distill(*_distill_inputs(7, 6, 2048, 20, ids, values), 0.7, 0.5, -3.0)


@pytest.mark.parametrize("V, stride", [(1000, 1008), (1001, 1008), (1001, 1003), (128256, 128264)])
def test_distill_loss_in_place_and_strided_rows(V, stride):
    """Rows with a stride of their own; the gradient in the logits' place, and in a buffer of another stride; what lies between the rows stays."""
    logits, tgt, ids, values = _distill_inputs(8, 5, V, 12)
    room = torch.full((5, stride), 7.0, dtype=bf, device="cuda")
    room[:, :V] = logits
    other = torch.full((5, stride + 5), 9.0, dtype=bf, device="cuda")
    first = _check_distill(room[:, :V], tgt, ids, values, 0.6, 2.0, 0.25, grad=other[:, :V])
    view = room[:, :V]
    second = _check_distill(view, tgt, ids, values, 0.6, 2.0, 0.25, grad=view)
    assert torch.equal(first[0], second[0]) and torch.equal(first[1], second[1])
    assert bool((room[:, V:] == 7).all()) and bool((other[:, V:] == 9).all())


def test_distill_loss_entries_that_repeat_or_do_not_exist():
    """Ids twice, the target among them, ids outside the vocabulary, values of minus infinity, rows without any entry."""
    logits, tgt, ids, values = _distill_inputs(3, 8, 500, 6)
    tgt[:] = torch.arange(8)
    ids[0] = 5
    ids[1, 3] = ids[1, 0]
    ids[2, 2:] = -1
    ids[3, 0], ids[3, 1] = 500, 2 ** 40
    ids[4] = -7
    values[5, 1:] = -math.inf
    values[6] = -math.inf
    ids[7, 0] = ids[7, 5] = 7
    values[4] = math.nan                 # entries that do not exist: their values are not used
    for weight in (0.5, 1.0):
        _check_distill(logits, tgt, ids, values, weight, 2.0, 1.0)


def test_distill_loss_masked_vocabulary():
    """Logits of minus infinity (a masked vocabulary) have no probability and no gradient."""
    logits, tgt, ids, values = _distill_inputs(4, 4, 20000, 5)
    keep = torch.zeros(4, 20000, dtype=torch.bool, device="cuda")
    keep.scatter_(1, ids, True).scatter_(1, tgt.clamp(0, 19999)[:, None], True)
    keep[:, 12345] = True
    logits.masked_fill_(~keep, -math.inf)
    _, grad = _check_distill(logits, tgt, ids, values, 0.4, 2.0, 1.0)
    assert not grad[~keep].any()


def test_distill_loss_without_rows_and_overlapping_gradients():
    from rocm_systems_b200.ops import train_ops

    logits, tgt, ids, values = _distill_inputs(5, 4, 64, 3)
    loss, grad = train_ops.distill_loss(logits[:0], tgt[:0], ids[:0], values[:0])
    assert loss.shape == (0,) and grad.shape == (0, 64)
    room = torch.zeros(4 * 64 + 64, dtype=bf, device="cuda")
    with pytest.raises(AssertionError, match="memory apart"):
        train_ops.distill_loss(room[:256].view(4, 64), tgt, ids, values, grad=room[64:].view(4, 64))
    with pytest.raises(AssertionError, match="one CUDA device"):
        train_ops.distill_loss(logits, tgt.cpu(), ids, values)


def test_distill_loss_repeats_bit_by_bit_and_in_a_graph():
    from rocm_systems_b200.ops import train_ops

    args = _distill_inputs(6, 50, 32000, 40)
    first = train_ops.distill_loss(*args, 0.5, 2.0, 0.1)
    assert all(torch.equal(a, b) for a, b in zip(first, train_ops.distill_loss(*args, 0.5, 2.0, 0.1)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = train_ops.distill_loss(*args, 0.5, 2.0, 0.1)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, kept))


# ---- together ------------------------------------------------------------------------------------------------------
def test_norms_rotation_and_attention_in_a_row():
    """The packed projection through both operators and back: each step's gradient is the next one's input, as in a layer."""
    from rocm_systems_b200.ops import attention, train_ops

    B, S, heads, kv, D, window, sinks = 2, 333, 6, 2, 64, 90, 4
    g = _gen(21)
    qkv = _rand(g, B, S, heads + 2 * kv, D).requires_grad_(True)
    wq, wk = ((1 + 0.2 * torch.randn(D, device="cuda", generator=g)).to(bf).requires_grad_(True) for _ in range(2))
    table = train_ops.rope_table(S, D, 500000.0, "cuda")
    q, k, v = attention.qk_norm_rope(qkv, wq, wk, table, heads, kv)
    out = attention.window_attention(q, k, v, window, sinks)
    dout = _rand(g, B, heads, S, D)
    mid = torch.autograd.grad(out, (q, k, v), dout, retain_graph=True)
    ref = oracle.attention(q, k, v, window, sinks, None, 1 / math.sqrt(D), dout)
    for n, t in zip(("out", "dq", "dk", "dv"), (out, *mid)):
        oracle.off(n, t, ref)
    back = torch.autograd.grad(out, (qkv, wq, wk), dout)
    ref = oracle.qk_norm_rope(qkv, wq, wk, table, heads, kv, 1e-5, mid)
    for n, t in zip(("dqkv", "dwq", "dwk"), back):
        oracle.off(n, t, ref)
    assert train_ops.gemm_take_error() == 0


def _big(*shape):
    return torch.empty(*shape, device="cuda", dtype=bf).normal_(generator=_gen(1))


def test_offsets_beyond_32_bits_attention():
    """The last sequence of a batch of more than 2^31 elements is what it is alone."""
    from rocm_systems_b200.ops import attention

    B, H, S, D = 2101, 8, 1024, 128
    q, dout = _big(B, S, H, D).transpose(1, 2), _big(B, S, H, D).transpose(1, 2)
    k, v = (_big(B, S, 1, D).transpose(1, 2) for _ in range(2))
    assert q.numel() > 2 ** 31
    lengths = torch.full((B,), S, device="cuda", dtype=torch.int32)
    lengths[-1] = 777

    def run(n):
        leaves = [t[n:].detach().requires_grad_(True) for t in (q, k, v)]
        out = attention.window_attention(*leaves, 300, 0, lengths[n:])
        return [t[-1] for t in (out, *torch.autograd.grad(out, leaves, dout[n:]))]

    for got, want in zip(run(0), run(B - 1)):
        assert torch.equal(got, want)


def test_offsets_beyond_32_bits_norms():
    from rocm_systems_b200.ops import attention, train_ops

    B, S, H, KV, D = 1030, 1024, 14, 1, 128
    qkv = _big(B, S, H + 2 * KV, D)
    assert qkv.numel() > 2 ** 31
    w = torch.ones(D, device="cuda", dtype=bf)
    table = train_ops.rope_table(S, D, 10000.0, "cuda")
    grads = [_big(S, n, D).transpose(0, 1).expand(B, n, S, D) for n in (H, KV, KV)]

    def run(n):
        x = qkv[n:].detach().requires_grad_(True)
        out = attention.qk_norm_rope(x, w, w, table, H, KV)
        dx, = torch.autograd.grad(out, (x,), [g[n:] for g in grads])
        return [t[-1] for t in (*out, dx)]

    for got, want in zip(run(0), run(B - 1)):
        assert torch.equal(got, want)


def test_offsets_beyond_32_bits_loss():
    from rocm_systems_b200.ops import train_ops

    T, V, K = 17000, 128256, 8
    logits = _big(T, V)
    assert logits.numel() > 2 ** 31
    tgt = torch.randint(0, V, (T,), device="cuda", generator=_gen(2))
    ids = torch.randint(0, V, (T, K), device="cuda", generator=_gen(3))
    values = torch.randn(T, K, device="cuda", generator=_gen(4))
    alone = train_ops.distill_loss(logits[-2:].clone(), tgt[-2:], ids[-2:], values[-2:], 0.5, 2.0, 0.125)
    loss, grad = train_ops.distill_loss(logits, tgt, ids, values, 0.5, 2.0, 0.125, grad=logits)
    assert torch.equal(loss[-2:], alone[0]) and torch.equal(grad[-2:], alone[1])


def test_calls_on_two_streams_at_once():
    """Each call has its own scratch: what runs beside it on another stream changes nothing."""
    from rocm_systems_b200.ops import attention, train_ops

    q, k, v, dout = _attention_inputs(5, 2, 8, 2, 900, 128)
    logits, tgt, ids, values = _distill_inputs(6, 64, 32000, 16)
    g = _gen(7)
    qkv, w = _rand(g, 2, 900, 12, 128).requires_grad_(True), torch.ones(128, device="cuda", dtype=bf).requires_grad_(True)
    table = train_ops.rope_table(900, 128, 10000.0, "cuda")

    def run():
        out = attention.window_attention(q, k, v, 200, 3)
        n = attention.qk_norm_rope(qkv, w, w, table, 8, 2)
        return [out, *torch.autograd.grad(out, (q, k, v), dout), *n, *torch.autograd.grad(n, (qkv, w), [torch.ones_like(t) for t in n]),
                *train_ops.distill_loss(logits, tgt, ids, values, 0.5, 2.5, 1.0)]

    want = run()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
