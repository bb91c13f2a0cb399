"""The student decoder's operators without a GPU: what they refuse, and the 64-bit oracles' gradients against differences."""
import pytest
import torch

import student_oracle as oracle

bf = torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _extension_built():
    from rocm_systems_b200.utils import build

    build.build_torch_ext()


def _qkv(**over):
    a = dict(B=2, S=8, heads=4, kv=2, D=64, dtype=bf)
    a |= over
    return torch.zeros(a["B"], a["S"], a["heads"] + 2 * a["kv"], a["D"], dtype=a["dtype"])


def _table(S=8, D=64):
    return torch.zeros(S, D // 2, 2)


def _w(D=64, dtype=bf):
    return torch.zeros(D, dtype=dtype)


@pytest.mark.parametrize("why, args", [
    ("in bf16", (_qkv(dtype=torch.float32), _w(), _w(), _table(), 4, 2)),
    ("in bf16", (_qkv()[0], _w(), _w(), _table(), 4, 2)),
    ("empty", (_qkv(S=0), _w(), _w(), _table(), 4, 2)),
    ("heads per token", (_qkv(), _w(), _w(), _table(), 4, 3)),
    ("heads per token", (_qkv(), _w(), _w(), _table(), 8, 0)),
    ("head dimension", (_qkv(D=60), _w(60), _w(60), _table(D=60), 4, 2)),
    ("head dimension", (_qkv(D=264), _w(264), _w(264), _table(D=264), 4, 2)),
    ("of one type", (_qkv(), _w(), _w(dtype=torch.float32), _table(), 4, 2)),
    ("of one type", (_qkv(), _w(32), _w(), _table(), 4, 2)),
    ("bf16 or fp32", (_qkv(), _w(dtype=torch.float16), _w(dtype=torch.float16), _table(), 4, 2)),
    ("at least S", (_qkv(), _w(), _w(), _table(7), 4, 2)),
    ("contiguous fp32", (_qkv(), _w(), _w(), _table().to(torch.float64), 4, 2)),
    ("eps", (_qkv(), _w(), _w(), _table(), 4, 2, float("nan"))),
    ("CUDA device", (_qkv(), _w(), _w(), _table(), 4, 2)),
])
def test_qk_norm_rope_refuses(why, args):
    from rocm_systems_b200.ops import attention

    with pytest.raises(AssertionError, match=why):
        attention.qk_norm_rope(*args)


def _t(B=2, H=4, S=8, D=64, dtype=bf):
    return torch.zeros(B, H, S, D, dtype=dtype)


@pytest.mark.parametrize("why, args, more", [
    ("q \\[B, H, S, D\\]", (_t()[0], _t(), _t()), {}),
    ("q \\[B, H, S, D\\]", (_t(), _t(H=2), _t()), {}),
    ("the same batch", (_t(), _t(S=9), _t(S=9)), {}),
    ("the same batch", (_t(), _t(B=1), _t(B=1)), {}),
    ("multiple of the key heads", (_t(), _t(H=3), _t(H=3)), {}),
    ("multiple of the key heads", (_t(S=0), _t(S=0), _t(S=0)), {}),
    ("head dimension", (_t(D=136), _t(D=136), _t(D=136)), {}),
    ("head dimension", (_t(D=4), _t(D=4), _t(D=4)), {}),
    ("bf16 tensors", (_t(dtype=torch.float16), _t(), _t()), {}),
    ("not negative", (_t(), _t(), _t()), {"window": -1}),
    ("not negative", (_t(), _t(), _t()), {"sinks": -1}),
    ("finite", (_t(), _t(), _t()), {"scale": float("nan")}),
    ("finite", (_t(), _t(), _t()), {"scale": -1.0}),
    ("int32", (_t(), _t(), _t()), {"lengths": torch.zeros(2, dtype=torch.int64)}),
    ("int32", (_t(), _t(), _t()), {"lengths": torch.zeros(3, dtype=torch.int32)}),
    ("CUDA device", (_t(), _t(), _t()), {}),
])
def test_window_attention_refuses(why, args, more):
    from rocm_systems_b200.ops import attention

    with pytest.raises(AssertionError, match=why):
        attention.window_attention(*args, **more)


def _loss_args(T=4, V=64, K=3, **over):
    a = {"logits": torch.zeros(T, V, dtype=bf), "targets": torch.zeros(T, dtype=torch.int64), "teacher_ids": torch.zeros(T, K, dtype=torch.int64),
         "teacher_logits": torch.zeros(T, K)}
    return a | over


@pytest.mark.parametrize("why, args", [
    ("in bf16 with dense rows", _loss_args(logits=torch.zeros(4, 64))),
    ("in bf16 with dense rows", _loss_args(logits=torch.zeros(64, 4, dtype=bf).t())),
    ("do not overlap", _loss_args(logits=torch.zeros(64, dtype=bf).expand(4, 64))),
    ("targets", _loss_args(targets=torch.zeros(4, dtype=torch.int32))),
    ("targets", _loss_args(targets=torch.zeros(5, dtype=torch.int64))),
    ("teacher_ids and teacher_logits", _loss_args(teacher_logits=torch.zeros(4, 2))),
    ("vocabulary", _loss_args(T=1, V=851969)),
    ("teacher entries", _loss_args(K=0)),
    ("teacher entries", _loss_args(K=1025)),
    ("int64 or int32 ids", _loss_args(teacher_ids=torch.zeros(4, 3, dtype=torch.int16))),
    ("int64 or int32 ids", _loss_args(teacher_logits=torch.zeros(4, 3, dtype=torch.float64))),
    ("temperature", _loss_args(temperature=0.0)),
    ("temperature", _loss_args(weight=1.5)),
    ("temperature", _loss_args(grad_scale=float("inf"))),
    ("like logits", _loss_args(grad=torch.zeros(4, 63, dtype=bf))),
    ("like logits", _loss_args(grad=torch.zeros(4, 64))),
    ("CUDA device", _loss_args()),
])
def test_distill_loss_refuses(why, args):
    from rocm_systems_b200.ops import train_ops

    with pytest.raises(AssertionError, match=why):
        train_ops.distill_loss(**args)


def test_c_entries_refuse_what_they_cannot_run():
    """The exported symbols check their numbers before anything is launched."""
    import ctypes

    from rocm_systems_b200 import _lib

    invalid = 1
    lib = _lib.load()
    vp, ll, i32, f32 = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int, ctypes.c_float
    lib.b200ops_qk_norm_rope_fwd.argtypes = [vp, vp, vp, i32, vp, vp, vp, ll] + [i32] * 4 + [f32, vp]
    lib.b200ops_qk_norm_rope_bwd.argtypes = [vp] * 7 + [i32] + [vp] * 5 + [ll] + [i32] * 4 + [f32, vp]
    lib.b200ops_window_attention_fwd.argtypes = [vp] * 8 + [i32] * 7 + [f32, vp]
    lib.b200ops_window_attention_bwd.argtypes = [vp] * 13 + [i32] * 7 + [f32, vp]
    lib.b200ops_distill_loss.argtypes = [vp, vp, vp, vp, i32, vp, i32, vp, ll, i32, i32, ll, ll, f32, f32, f32, vp]
    none = (ctypes.c_longlong * 24)()
    p = 4096  # an address that nothing reads: every call below is refused
    fwd = lambda B=1, H=2, KV=1, S=4, D=64, w=0, si=0, q=p: lib.b200ops_window_attention_fwd(q, p, p, p, None, None, None, none, B, H, KV, S, D, w, si, 1.0, None)
    for bad in ({"B": 0}, {"H": 0}, {"KV": 0}, {"H": 3, "KV": 2}, {"S": 0}, {"D": 136}, {"D": 20}, {"D": 0}, {"w": -1}, {"si": -1}, {"q": p + 2}, {"q": None}):
        assert fwd(**bad) == invalid, bad
    assert lib.b200ops_window_attention_fwd(p, p, p, p, None, None, None, none, 1, 2, 1, 4, 64, 0, 0, -1.0, None) == invalid
    odd = (ctypes.c_longlong * 24)(*([4] * 24))
    assert lib.b200ops_window_attention_fwd(p, p, p, p, None, None, None, odd, 1, 2, 1, 4, 64, 0, 0, 1.0, None) == invalid
    assert lib.b200ops_window_attention_bwd(p, p, p, p, p, p, None, p, p, p, p, None, none, 1, 2, 1, 4, 64, 0, 0, 1.0, None) == invalid
    assert lib.b200ops_window_attention_bwd(p, p, p, p, p, p + 8, p, p, p, p, p, None, none, 1, 2, 1, 4, 64, 0, 0, 1.0, None) == invalid
    for seq, heads, kv, D in ((0, 4, 2, 64), (8, 0, 2, 64), (8, 4, 0, 64), (8, 4, 2, 12), (8, 4, 2, 512)):
        assert lib.b200ops_qk_norm_rope_fwd(p, p, p, 1, p, p, p, 8, seq, heads, kv, D, 1e-5, None) == invalid
        assert lib.b200ops_qk_norm_rope_bwd(p, p, p, none, p, p, p, 1, p, p, p, p, p, 8, seq, heads, kv, D, 1e-5, None) == invalid
    loss = lambda T=4, V=64, K=3, st=64, gst=64, ib=8, vb=4, tau=1.0: lib.b200ops_distill_loss(p, p, p, p, ib, p, vb, p, T, V, K, st, gst, 1.0, tau, 1.0, None)
    for bad in ({"T": -1}, {"V": 0}, {"V": 851969, "st": 851976, "gst": 851976}, {"K": 0}, {"K": 1025}, {"st": 63}, {"gst": 8}, {"ib": 2}, {"vb": 8}, {"tau": 0.0}, {"tau": float("nan")}):
        assert loss(**bad) == invalid, bad


def test_oracle_gradients_are_those_of_the_definitions():
    """The oracles' gradients against automatic differentiation and, through it, differences."""
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    q, k, v, do = r(2, 4, 9, 8), r(2, 2, 9, 8), r(2, 2, 9, 8), r(2, 4, 9, 8)
    lengths = torch.tensor([9, 5], dtype=torch.int32)

    def attn(q, k, v):
        s = q @ k.repeat_interleave(2, 1).transpose(-1, -2) * 0.4
        i = torch.arange(9)
        see = (i[None, :] <= i[:, None]) & ((i[:, None] - i[None, :] < 3) | (i[None, :] < 2))
        p = torch.softmax(s.masked_fill(~see, float("-inf")), -1) @ v.repeat_interleave(2, 1)
        return p * (i < lengths.view(2, 1)).view(2, 1, 9, 1)

    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    assert torch.autograd.gradcheck(attn, leaves)
    ref = oracle.attention(q, k, v, 3, 2, lengths, 0.4, do)
    assert torch.allclose(attn(*leaves), ref["out"])
    for n, t in zip(("dq", "dk", "dv"), torch.autograd.grad(attn(*leaves), leaves, do)):
        assert torch.allclose(t, ref[n]), n

    x, wq, wk = (t.requires_grad_(True) for t in (r(2, 5, 4, 8), r(8), r(8)))
    ang = r(5, 4)
    table = torch.stack([ang.cos(), ang.sin()], -1)
    grads = r(2, 2, 5, 8), r(2, 1, 5, 8), r(2, 1, 5, 8)

    def norm(x, wq, wk):
        def one(t, w):
            n = t / (t.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w
            c = torch.view_as_complex(torch.stack([n[..., :4], n[..., 4:]], -1)) * torch.complex(table[..., 0], table[..., 1])[:, None]
            return torch.cat([c.real, c.imag], -1).transpose(1, 2)
        return one(x[:, :, :2], wq), one(x[:, :, 2:3], wk), x[:, :, 3:].transpose(1, 2)

    assert torch.autograd.gradcheck(norm, (x, wq, wk))
    ref = oracle.qk_norm_rope(x, wq, wk, table, 2, 1, 1e-5, grads)
    for n, t in zip(("q", "k", "v"), norm(x, wq, wk)):
        assert torch.allclose(t, ref[n]), n
    for n, t in zip(("dqkv", "dwq", "dwk"), torch.autograd.grad(norm(x, wq, wk), (x, wq, wk), grads)):
        assert torch.allclose(t, ref[n]), n

    z = r(3, 11).requires_grad_(True)
    ids, values, tgt = torch.tensor([[1, 4, 4], [0, 10, 3], [2, 5, 6]]), r(3, 3), torch.tensor([4, 7, -1])

    def loss(z):
        logp, logq = torch.log_softmax(values / 2, 1), torch.log_softmax(z / 2, 1).gather(1, ids)
        rows = 0.3 * 4 * (logp.exp() * (logp - logq)).sum(1) - 0.7 * torch.log_softmax(z, 1).gather(1, tgt.clamp(min=0)[:, None])[:, 0]
        return rows * (tgt >= 0)

    assert torch.autograd.gradcheck(loss, (z,))
    ref = oracle.distill(z, tgt, ids, values, 0.3, 2.0, 0.5)
    assert torch.allclose(loss(z), ref["loss"])
    assert torch.allclose(torch.autograd.grad(loss(z).sum(), z)[0] * 0.5, ref["grad"])


@pytest.mark.parametrize("B, H, KV, S, D, window, sinks", [(1, 32, 8, 4096, 128, 1024, 4), (1, 32, 8, 131072, 128, 1024, 131072), (1, 32, 8, 131072, 128, 128, 4096),
                                                           (4, 32, 8, 8192, 128, 128, 2000), (64, 32, 8, 8192, 64, 1, 300), (1, 1, 1, 1 << 20, 128, 1, 1)])
def test_window_attention_backward_scratch_is_bounded(B, H, KV, S, D, window, sinks):
    """However many sinks there are: rows' statistics, and at most 2048 blocks of 128 rows of two gradients for the sinks' partial sums."""
    import ctypes

    from rocm_systems_b200 import _lib

    words = _lib.load().b200ops_window_attention_bwd_scratch
    words.argtypes, words.restype = [ctypes.c_int] * 7, ctypes.c_longlong
    stats = B * H * ((S + 127) // 128 * 128) * 4
    assert stats <= words(B, H, KV, S, D, window, sinks) <= stats + 2048 * 2 * 128 * D


@pytest.mark.parametrize("temperature", [1e-45, 1e-6, 0.0099, 101.0, 1e6, 1e30, float("nan")])
def test_distill_loss_refuses_temperatures_beyond_its_arithmetic(temperature):
    """Scores are scaled by 1 / temperature in fp32, and the divergence by its square."""
    from rocm_systems_b200.ops import train_ops

    with pytest.raises(AssertionError, match="temperature"):
        train_ops.distill_loss(**_loss_args(temperature=temperature))
