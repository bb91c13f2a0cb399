"""What the student decoder's operators refuse of autograd, and what their native library says about itself, without a GPU."""
import pytest
import torch

bf = torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _extension_built():
    from rocm_systems_b200.utils import build

    build.build_torch_ext()


def _norm_args(**over):
    a = {"qkv": torch.zeros(2, 8, 8, 64, dtype=bf), "q_weight": torch.zeros(64, dtype=bf), "k_weight": torch.zeros(64, dtype=bf), "table": torch.zeros(8, 32, 2),
         "heads": 4, "kv_heads": 2}
    return a | over


def _attention_args():
    return {n: torch.zeros(2, 4, 8, 64, dtype=bf) for n in "qkv"}


def _loss_args():
    return {"logits": torch.zeros(4, 64, dtype=bf), "targets": torch.zeros(4, dtype=torch.int64), "teacher_ids": torch.zeros(4, 3, dtype=torch.int64),
            "teacher_logits": torch.zeros(4, 3), "weight": 0.5}


@pytest.mark.parametrize("op, args, dual", [
    *(("qk_norm_rope", _norm_args, n) for n in ("qkv", "q_weight", "k_weight", "table")),
    *(("window_attention", _attention_args, n) for n in "qkv"),
    *(("distill_loss", _loss_args, n) for n in ("logits", "teacher_logits")),
])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(op, args, dual, grad):
    """A dual tensor does not require a gradient, and its tangent would be dropped."""
    from torch.autograd import forward_ad

    from rocm_systems_b200.ops import attention, train_ops

    call, args = getattr(attention, op, None) or getattr(train_ops, op), args()
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        args[dual] = forward_ad.make_dual(args[dual], torch.ones_like(args[dual]))
        with pytest.raises(AssertionError, match="forward-mode"):
            call(**args)


def test_a_table_that_asks_for_a_gradient_is_refused():
    from rocm_systems_b200.ops import attention

    args = _norm_args(table=torch.zeros(8, 32, 2, requires_grad=True))
    with pytest.raises(AssertionError, match="table: a gradient"):
        attention.qk_norm_rope(**args)
    with torch.no_grad(), pytest.raises(AssertionError, match="CUDA device"):  # nothing but the device is wrong
        attention.qk_norm_rope(**args)


@pytest.mark.parametrize("S, window, sinks, launches", [(900, 0, 0, 2), (900, 100, 0, 2), (900, 100, 3, 3), (900, 0, 3, 2), (900, 900, 3, 2), (200, 100, 3, 2), (1, 1, 1, 2),
                                                        (900, 100, 900, 2)])
def test_window_attention_says_how_many_kernels_a_backward_call_launches(S, window, sinks, launches):
    import ctypes

    from rocm_systems_b200 import _lib

    args = (1, 2, 1, S, 64, window, sinks)
    count, words = _lib.load().b200ops_window_attention_bwd_launches, _lib.load().b200ops_window_attention_bwd_scratch
    count.argtypes, words.argtypes, words.restype = [ctypes.c_int] * 7, [ctypes.c_int] * 7, ctypes.c_longlong
    assert count(*args) == launches
    assert (words(*args) > 2 * ((S + 127) // 128 * 128) * 4) == (launches == 3)  # partial sums, and the kernel that adds them up
    assert count(1, 2, 1, S, 60, window, sinks) == -1
