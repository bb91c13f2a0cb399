"""The student decoder's operators where their variants meet: padded batches and odd head dimensions beyond the shortest sequences, values that
are not finite, small losses, what autograd may do with a call."""
import math

import pytest
import torch

import student_oracle as oracle

pytestmark = pytest.mark.gpu
bf = torch.bfloat16
NAMES = ("out", "dq", "dk", "dv")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rand(g, *shape, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(bf)


def _inputs(seed, B, H, KV, S, D):
    g = _gen(seed)
    packed = _rand(g, B, S, H + 2 * KV, D)
    q, k, v = (packed[:, :, a:b].transpose(1, 2).detach() for a, b in ((0, H), (H, H + KV), (H + KV, H + 2 * KV)))
    return q, k, v, _rand(g, B, S, H, D).transpose(1, 2)


def _both_ways(q, k, v, dout, window=0, sinks=0, lengths=None):
    from rocm_systems_b200.ops import attention

    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = attention.window_attention(q, k, v, window, sinks, lengths)
    return dict(zip(NAMES, (out.detach(), *torch.autograd.grad(out, (q, k, v), dout))))


def _against_the_oracle(q, k, v, dout, window, sinks, lengths=None):
    got = _both_ways(q, k, v, dout, window, sinks, lengths)
    ref = oracle.attention(q, k, v, window, sinks, lengths, 1 / math.sqrt(q.shape[-1]), dout)
    for n in NAMES:
        oracle.off(n, got[n], ref)
    return got


# ---- how weights are rounded -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [0, 40, 64, 65, 300])
def test_padding_changes_no_bit_of_a_sequence(D, window):
    """A sequence in a padded batch has the answer and the gradients that it has alone, however long the others are."""
    lengths = (700, 3, 130, 256, 257, 1, 0)
    q, k, v, dout = _inputs(7, len(lengths), 4, 2, 700, D)
    got = _both_ways(q, k, v, dout, window, 0, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        alone = _both_ways(*(t[b:b + 1, :, :n] for t in (q, k, v, dout)), window)
        for name in NAMES:
            assert torch.equal(got[name][b:b + 1, :, :n], alone[name]), (name, n)


@pytest.mark.parametrize("S, window, sinks", [(300, 0, 0), (700, 0, 0), (700, 200, 5), (1100, 70, 150)])
@pytest.mark.parametrize("D", [64, 128])
def test_a_long_sequences_first_rows_are_as_exact_as_a_short_one(S, D, window, sinks):
    """Their gradient is a difference of few weights. Answers and gradients of the first 128 rows do not depend on what follows; the keys' gradients do
    not where the later rows' gradient is zero. So the bounds of a sequence of 128 tokens hold."""
    q, k, v, dout = _inputs(S + D, 2, 4, 2, S, D)
    q = q * 2
    dout = torch.where(torch.arange(S, device="cuda").view(S, 1) < 128, dout, torch.zeros_like(dout))
    got = _both_ways(q, k, v, dout, window, sinks)
    ref = oracle.attention(*(t[:, :, :128] for t in (q, k, v)), window, sinks, None, 1 / math.sqrt(D), dout[:, :, :128])
    for n in NAMES:
        oracle.off(n, got[n][:, :, :128], ref)
    assert not got["dk"][:, :, 128:].any() and not got["dv"][:, :, 128:].any()


# ---- values that are not finite ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("S, D", [(200, 64), (500, 64), (500, 128)])
def test_window_attention_a_key_that_is_not_a_number(S, D):
    """Rows that see it answer NaN, whichever of a tile's columns it is in; the others do not notice."""
    B = 128
    q, k, v, dout = _inputs(S, B, 1, 1, S, D)
    at = torch.arange(B, device="cuda")
    k[at, 0, at, 5] = math.nan
    got = _both_ways(q, k, v, dout)
    sees = torch.arange(S, device="cuda")[None, :] >= at[:, None]
    assert bool(torch.isnan(got["out"][:, 0][sees]).all()) and bool(torch.isfinite(got["out"][:, 0][~sees]).all())
    assert bool(torch.isnan(got["dq"][:, 0][sees]).all())
    assert bool(torch.isnan(got["dk"]).all()) and bool(torch.isnan(got["dv"]).all())  # the last row sees all of them


def test_window_attention_a_key_that_is_infinite():
    """A score of plus infinity leaves no number; one of minus infinity is a key that counts nothing."""
    B, S, D = 128, 500, 64
    q, k, v, dout = _inputs(3, B, 1, 1, S, D)
    at = torch.arange(B, device="cuda")
    k[at, 0, at, 0] = math.inf
    sign = torch.where(torch.rand(B, S, device="cuda", generator=_gen(1)) < 0.5, 1.0, -1.0)
    q[:, 0, :, 0] = sign.to(bf)
    out = _both_ways(q, k, v, dout)["out"][:, 0]
    rows = torch.arange(S, device="cuda")
    sees = rows[None, :] >= at[:, None]
    nothing = (at[:, None] == 0) & (rows[None, :] == 0)  # no other key
    bad = (sees & (sign > 0)) | nothing
    assert bool(torch.isnan(out[bad]).all())
    k[at, 0, at, 0] = 0
    scores = q[:, 0].double() @ k[:, 0].double().transpose(1, 2) / math.sqrt(D)
    scores.masked_fill_(rows[None, :] > rows[:, None], -math.inf)
    scores[at, :, at] = -math.inf
    P = torch.softmax(scores, -1)
    # every weight is rounded to bf16 and the answer again; the scores' own errors are far smaller
    tol = 2.0 ** -8 * (P @ v[:, 0].double()).abs() + (2.0 ** -8 + 2.0 ** -12) * (P @ v[:, 0].double().abs())
    good = sees & ~bad
    assert bool(((out.double() - P @ v[:, 0].double()).abs() <= tol)[good].all())


@pytest.mark.parametrize("S", [100, 700])
def test_window_attention_rows_of_nothing_but_minus_infinity(S):
    """Rows all of whose visible scores are minus infinity have no softmax."""
    q, k, v, _ = _inputs(5, 1, 2, 1, S, 64)
    k[..., 0] = -k[..., 0].abs() - 0.5
    q[0, 1, S // 2:, 0] = math.inf
    from rocm_systems_b200.ops import attention

    out = attention.window_attention(q, k, v)
    assert bool(torch.isnan(out[0, 1, S // 2:]).all()) and bool(torch.isfinite(out[0, 0]).all()) and bool(torch.isfinite(out[0, 1, :S // 2]).all())


@pytest.mark.parametrize("K", [1, 5, 40])
def test_distill_loss_a_teacher_that_is_not_a_number(K):
    """It is not a row without entries: the loss, and the gradient of the entries' logits, are not numbers either."""
    from rocm_systems_b200.ops import train_ops

    g = _gen(K)
    logits, tgt = _rand(g, 4, 300), torch.arange(4, device="cuda")
    ids = torch.stack([torch.randperm(300, device="cuda", generator=g)[:K] for _ in range(4)])
    values = torch.randn(4, K, device="cuda", generator=g)
    values[1] = math.nan
    values[2, K - 1] = math.nan
    values[3] = -math.inf      # entries of no weight: a row without any
    for weight in (0.5, 1.0):
        loss, grad = train_ops.distill_loss(logits, tgt, ids, values, weight, 2.0)
        assert torch.isnan(loss).tolist() == [False, True, True, False]
        assert torch.isnan(grad.gather(1, ids)).all(-1).tolist() == [False, True, True, False] and bool(torch.isfinite(grad[[0, 3]]).all())


@pytest.mark.parametrize("weight, tau", [(0.0, 1.0), (0.0, 3.0), (1.0, 1.0), (1.0, 0.01), (1.0, 0.1), (0.5, 1.0), (0.5, 2.0), (0.5, 3.0), (0.5, 4.0), (0.5, 2.5), (0.5, 0.1)])
@pytest.mark.parametrize("V", [500, 40000])
def test_distill_loss_small_losses_of_large_logits(V, weight, tau):
    """A student that is all but sure of what target and teacher say: the loss is the logarithm of a sum that hardly differs from one.

    Each power of two is off by 2^-22 of itself, of the largest one that is the sum's error, once more where the slices' sums are joined; the logarithm adds
    2^-23: below 2^-20 together, of each softmax. Nothing of it grows with the logits' size."""
    from rocm_systems_b200.ops import train_ops

    tops = torch.cat([torch.arange(16, 32, 0.125), torch.arange(32, 128, 0.5)]).to("cuda")
    T = tops.numel()
    g = _gen(V)
    logits = _rand(g, T, V, scale=0.5)
    tgt = torch.randint(0, V, (T,), device="cuda", generator=g)
    logits[torch.arange(T), tgt] = tops.to(bf)
    loss, _ = train_ops.distill_loss(logits, tgt, tgt[:, None].contiguous(), torch.zeros(T, 1, device="cuda"), weight, tau)
    z = logits.double()
    ce, kl = (-torch.log_softmax(z / t, -1).gather(1, tgt[:, None])[:, 0] for t in (1.0, tau))
    want = (1 - weight) * ce + weight * tau ** 2 * kl
    # sums over the row: one rounding per addition of a thread (128 of them side by side in each of up to 8 slices) and of the tree behind them
    seq = (V / 128 + 16) * 2.0 ** -24
    tol = (1 - weight) * (2.0 ** -20 + seq * ce) + weight * tau ** 2 * (2.0 ** -20 + seq * kl) + 2.0 ** -18 * want
    over = (loss.double() - want).abs() - tol
    assert bool((over <= 0).all()), (float(over.max()), float(want[over.argmax()]), float(tops[over.argmax()]))


@pytest.mark.parametrize("loss", ["distill", "cross_entropy"])
def test_a_gradient_in_the_logits_place_is_seen_by_autograd(loss):
    """A graph that saved the logits refuses its backward pass once the gradient has taken their place."""
    from rocm_systems_b200.ops import train_ops

    x = _rand(_gen(1), 4, 64).requires_grad_(True)
    tgt, ids, values = torch.arange(4, device="cuda"), torch.zeros(4, 1, dtype=torch.int64, device="cuda"), torch.zeros(4, 1, device="cuda")
    logits = x * 2
    other = logits.square().sum()  # keeps the logits
    version = logits._version
    with torch.no_grad():
        if loss == "distill":
            train_ops.distill_loss(logits, tgt, ids, values, 0.5, 2.0)
            assert logits._version == version
            train_ops.distill_loss(logits, tgt, ids, values, 0.5, 2.0, grad=logits)
        else:
            train_ops.cross_entropy_inplace(logits, tgt, 1.0)
    assert logits._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        other.backward()
    with torch.inference_mode():  # tensors without versions
        plain = torch.zeros(4, 64, dtype=bf, device="cuda")
        train_ops.distill_loss(plain, tgt, ids, values, 0.5, 2.0, grad=plain)
        train_ops.cross_entropy_inplace(plain, tgt, 1.0)


def _norm_inputs(seed, B=2, S=37, heads=4, kv=2, D=64, weights=bf):
    from rocm_systems_b200.ops import train_ops

    g = _gen(seed)
    qkv = _rand(g, B, S, heads + 2 * kv, D)
    w = [(1 + 0.3 * torch.randn(D, device="cuda", generator=g)).to(weights) for _ in range(2)]
    grads = tuple(_rand(g, B, S, n, D).transpose(1, 2) for n in (heads, kv, kv))
    return (qkv, *w), train_ops.rope_table(S, D, 10000.0, "cuda"), grads

def test_launches_are_counted():
    from rocm_systems_b200.ops import attention, train_ops

    def count(fn):
        before = attention.launches()
        fn()
        return attention.launches() - before

    q, k, v, dout = _inputs(2, 1, 2, 1, 900, 64)
    assert count(lambda: attention.window_attention(q, k, v, 100, 3)) == 1
    assert count(lambda: _both_ways(q, k, v, dout)) == 3
    assert count(lambda: _both_ways(q, k, v, dout, 100, 3)) == 4      # the sinks' sums are joined
    assert count(lambda: _both_ways(q, k, v, dout, 100, 0)) == 3
    inputs, table, grads = _norm_inputs(1)
    leaf = inputs[0].detach().requires_grad_(True)
    assert count(lambda: attention.qk_norm_rope(*inputs, table, 4, 2)) == 1
    assert count(lambda: torch.autograd.grad(attention.qk_norm_rope(leaf, *inputs[1:], table, 4, 2), leaf, grads)) == 3
    logits, tgt, ids, values = _rand(_gen(1), 3, 64), torch.arange(3, device="cuda"), torch.zeros(3, 1, dtype=torch.int64, device="cuda"), torch.zeros(3, 1, device="cuda")
    assert count(lambda: train_ops.distill_loss(logits, tgt, ids, values)) == 1
    assert count(lambda: train_ops.distill_loss(logits[:0], tgt[:0], ids[:0], values[:0])) == 0


# ---- what autograd may do with a call -----------------------------------------------------------------------------------
def test_gradients_of_gradients_are_refused():
    from rocm_systems_b200.ops import attention

    q, k, v, dout = _inputs(1, 1, 2, 1, 20, 64)
    q.requires_grad_(True)
    with pytest.raises(RuntimeError, match="not itself differentiable"):
        torch.autograd.grad(attention.window_attention(q, k, v), q, dout, create_graph=True)
    (qkv, wq, wk), table, grads = _norm_inputs(2)
    qkv.requires_grad_(True)
    with pytest.raises(RuntimeError, match="not itself differentiable"):
        torch.autograd.grad(attention.qk_norm_rope(qkv, wq, wk, table, 4, 2), qkv, grads, create_graph=True)


@pytest.mark.parametrize("S, window, sinks", [(150, 0, 0), (500, 90, 3)])
@pytest.mark.parametrize("which", [(0,), (1,), (2,), (0, 2)])
def test_a_gradient_of_some_inputs_only(S, window, sinks, which):
    """The same bits as when all of them need one."""
    from rocm_systems_b200.ops import attention

    q, k, v, dout = _inputs(S, 2, 4, 2, S, 64)
    want = _both_ways(q, k, v, dout, window, sinks)
    leaves = [t.detach().requires_grad_(i in which) for i, t in enumerate((q, k, v))]
    got = torch.autograd.grad(attention.window_attention(*leaves, window, sinks), [leaves[i] for i in which], dout)
    for i, t in zip(which, got):
        assert torch.equal(t, want[("dq", "dk", "dv")[i]])


@pytest.mark.parametrize("which", [(0,), (1,), (2,), (0, 1)])
def test_norms_a_gradient_of_some_inputs_only(which):
    from rocm_systems_b200.ops import attention

    inputs, table, grads = _norm_inputs(3)

    def run(which):
        leaves = [t.detach().requires_grad_(i in which) for i, t in enumerate(inputs)]
        return torch.autograd.grad(attention.qk_norm_rope(*leaves, table, 4, 2), [leaves[i] for i in which], grads)

    want = run((0, 1, 2))
    assert all(torch.equal(t, want[i]) for i, t in zip(which, run(which)))


# ---- padded batches and head dimensions beyond 256 tokens ----------------------------------------------------------------
@pytest.mark.parametrize("lengths", [(700, 0, 1, 3), (127, 129, 700, 400), (257, 512, 640, 641)])
@pytest.mark.parametrize("D, window, sinks", [(64, 0, 0), (96, 0, 0), (128, 0, 0), (64, 100, 4), (128, 100, 4), (72, 130, 140), (128, 130, 140), (96, 300, 600)])
def test_padded_batches_of_longer_sequences(lengths, D, window, sinks):
    """As for the short ones: NaN and infinities behind a sequence's end are not used; its rows answer zeros and get zero gradients, also where the
    sinks' later queries are split and a sequence ends before them or among the sinks."""
    S = 700
    q, k, v, dout = _inputs(D + window, 4, 4, 2, S, D)
    L = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for t in (q, k, v, dout):
        for b, n in enumerate(lengths):
            t[b, :, n:] = math.nan
            t[b, :, n:, ::3] = math.inf
    got = _against_the_oracle(q, k, v, dout, window, sinks, L)
    for n, t in got.items():
        for b, m in enumerate(lengths):
            assert not t[b, :, m:].any(), n


@pytest.mark.parametrize("lengths", [(1100, 3), (130, 1099), (0, 513)])
@pytest.mark.parametrize("D, window, sinks", [(128, 100, 4), (64, 65, 300), (40, 0, 0)])
def test_padded_batches_of_long_sequences(lengths, D, window, sinks):
    S = 1100
    q, k, v, dout = _inputs(D + window, 2, 2, 1, S, D)
    L = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for t in (q, k, v, dout):
        for b, n in enumerate(lengths):
            t[b, :, n:] = math.nan
    got = _against_the_oracle(q, k, v, dout, window, sinks, L)
    for n, t in got.items():
        for b, m in enumerate(lengths):
            assert not t[b, :, m:].any(), n


@pytest.mark.parametrize("B, H, KV, D", [(1, 1, 1, 8), (2, 3, 1, 128), (1, 4, 4, 104), (2, 6, 2, 96), (1, 8, 1, 40), (3, 2, 2, 16), (1, 5, 5, 72), (1, 7, 1, 120)])
@pytest.mark.parametrize("S, window, sinks", [(400, 0, 0), (400, 90, 5), (641, 129, 1)])
def test_head_dimensions_of_longer_sequences(B, H, KV, D, S, window, sinks):
    _against_the_oracle(*_inputs(S + D, B, H, KV, S, D), window, sinks)


@pytest.mark.parametrize("D", [64, 72, 128])
def test_layouts_of_longer_sequences(D):
    """Heads outside positions, rows off 16 bytes, one key head's memory for all, a transposed gradient, a gradient that is one number."""
    B, H, KV, S = 2, 4, 2, 450
    g = _gen(D)
    q = _rand(g, B, H, S, D)
    k = _rand(g, B * KV * S * D + 1)[1:].view(B, KV, S, D)
    v = _rand(g, B, 1, S, D).expand(B, KV, S, D)
    _against_the_oracle(q, k, v, _rand(g, B, H, D, S).transpose(2, 3), 133, 2)
    _against_the_oracle(_rand(g, B, S, H, D + 8)[..., :D].transpose(1, 2), k, v, _rand(g, 1, 1, 1, 1).expand(B, H, S, D), 0, 0)


def _elsewhere(t):
    """The same values in other memory: dimensions in another order, every row off its 16 bytes."""
    if t.dim() < 2:
        return torch.cat([t[:1], t])[1:]
    room = torch.empty(tuple(reversed(t.shape[:-1])) + (t.shape[-1] + 1,), dtype=t.dtype, device=t.device)
    room = room[..., 1:].permute(*reversed(range(t.dim() - 1)), t.dim() - 1)
    return room.copy_(t)


@pytest.mark.parametrize("unpack", [lambda t: t.clone(memory_format=torch.contiguous_format), _elsewhere])
def test_saved_tensors_may_come_back_in_other_memory(unpack):
    """A hook on saved tensors gives back equal values; where and in which order they lie is its own affair."""
    from rocm_systems_b200.ops import attention

    q, k, v, dout = _inputs(9, 2, 4, 2, 300, 64)
    inputs, table, grads = _norm_inputs(4)
    L = torch.tensor([300, 170], dtype=torch.int32, device="cuda")

    def run():
        a = [t.detach().requires_grad_(True) for t in (q, k, v)]
        b = [t.detach().requires_grad_(True) for t in inputs]
        out, normed = attention.window_attention(*a, 90, 3, L), attention.qk_norm_rope(*b, table, 4, 2)
        return [*torch.autograd.grad(out, a, dout), *torch.autograd.grad(normed, b, grads)]

    want = run()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: unpack(t)):
        got = run()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_saved_tensors_kept_on_the_host():
    from rocm_systems_b200.ops import attention

    q, k, v, dout = _inputs(9, 2, 4, 2, 300, 64)
    want = _both_ways(q, k, v, dout, 90, 3)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    with torch.autograd.graph.save_on_cpu():
        out = attention.window_attention(*leaves, 90, 3)
    for n, t in zip(NAMES[1:], torch.autograd.grad(out, leaves, dout)):
        assert torch.equal(t, want[n]), n


def test_saved_tensors_that_are_something_else_are_refused():
    from rocm_systems_b200.ops import attention

    q, k, v, dout = _inputs(9, 1, 2, 1, 40, 64)
    inputs, table, grads = _norm_inputs(4)
    for change in (lambda t: t.float() if t.dtype == bf else t.double() if t.dtype == torch.float32 else t, lambda t: t.cpu(), lambda t: t[..., :-1]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            a, b = q.detach().requires_grad_(True), inputs[0].detach().requires_grad_(True)
            out, normed = attention.window_attention(a, k, v), attention.qk_norm_rope(b, *inputs[1:], table, 4, 2)
        with pytest.raises(RuntimeError, match="saved"):
            torch.autograd.grad(out, a, dout)
        with pytest.raises(RuntimeError, match="saved"):
            torch.autograd.grad(normed, b, grads)


@pytest.mark.parametrize("S, window, sinks", [(1, 0, 0), (1, 1, 1), (5, 1, 0), (130, 1, 0), (700, 1, 0)])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_that_see_one_key_have_no_gradient_of_scores(S, window, sinks, D):
    """Their one weight is one whatever the score is. Not even rounding noise is left of a difference that is zero by definition."""
    q, k, v, dout = _inputs(S, 2, 4, 2, S, D)
    got = _against_the_oracle(q, k, v, dout, window, sinks)
    assert not got["dq"].any() and not got["dk"].any()


@pytest.mark.parametrize("S, window, sinks", [(2, 0, 0), (300, 1, 1), (300, 0, 0), (700, 90, 5)])
def test_a_sequences_first_row_sees_one_key(S, window, sinks):
    q, k, v, dout = _inputs(S, 2, 4, 2, S, 64)
    first = torch.zeros_like(dout)
    first[:, :, 0] = dout[:, :, 0]
    got = _both_ways(q, k, v, first, window, sinks)
    assert not got["dq"].any() and not got["dk"].any()
    q[0, 0, 0, 0] = math.nan
    assert bool(torch.isnan(_both_ways(q, k, v, first, window, sinks)["dq"][0, 0, 0]).all())


@pytest.mark.parametrize("weight, tau", [(0.0, 1.0), (1.0, 1.0), (1.0, 0.01), (1.0, 100.0), (0.5, 1.0), (0.5, 2.0), (0.5, 3.0), (0.5, 4.0), (0.5, 2.5), (0.5, 0.1)])
@pytest.mark.parametrize("V", [500, 40000])
def test_distill_loss_logits_up_to_a_hundred_million_temperatures(V, weight, tau):
    """Two equal logits far above all others: a half each. The rounding of so large an offset is a factor of up to 16 of every power; it is taken out."""
    from rocm_systems_b200.ops import train_ops

    tops = (torch.logspace(1, 8, 300, device="cuda") * min(tau, 1.0)).clamp(min=3000 * max(tau, 1.0)).to(bf)
    T = tops.numel()
    g = _gen(V)
    for sign in (1, -1):  # the others at zero, or the two at zero and the others far below
        logits = torch.zeros(T, V, dtype=bf, device="cuda")
        tgt = torch.randint(0, V // 2, (T,), device="cuda", generator=g)
        two = torch.stack([tgt, tgt + V // 2], 1)  # in two slices where there are several
        if sign > 0:
            logits.scatter_(1, two, tops[:, None].expand(T, 2).contiguous())
        else:
            logits[:] = -tops[:, None]
            logits.scatter_(1, two, 0)
        loss, grad = train_ops.distill_loss(logits, tgt, tgt[:, None].contiguous(), torch.zeros(T, 1, device="cuda"), weight, tau)
        want = (1 - weight + weight * tau ** 2) * math.log(2)
        # as for small losses, and the rounding of the loss
        assert float((loss.double() - want).abs().max()) <= (1 - weight + weight * tau ** 2) * (2.0 ** -20 + (V / 128 + 16) * 2.0 ** -24 + 2.0 ** -22)
        dense = torch.zeros(T, V, dtype=torch.float64, device="cuda")
        dense.scatter_(1, two, (1 - weight + weight * tau) * torch.tensor([[-0.5, 0.5]], dtype=torch.float64, device="cuda").expand(T, 2).contiguous())
        assert float((grad.double() - dense).abs().max()) <= (1 - weight + weight * tau) * (0.5 * 2.0 ** -8 + 2.0 ** -18)
