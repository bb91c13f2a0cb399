"""A student decoder's training step: per-head norms, windowed attention with sinks and a teacher's logits together in the trainer."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _reference(cfg, weights, tok, tgt, ids, values, distill, dtype=torch.float64):
    """Loss and gradients of the same decoder by automatic differentiation in 64 bits."""
    d, nh, nkv = cfg.head_dim, cfg.heads, cfg.kv_heads
    W = {k: v.detach().to(dtype).requires_grad_(True) for k, v in weights.items()}
    B, S = tok.shape
    inv = 1.0 / (cfg.rope_theta ** (torch.arange(0, d, 2, device=tok.device, dtype=torch.float64) / d))
    ang = torch.outer(torch.arange(S, device=tok.device, dtype=torch.float64), inv)
    turn = torch.complex(ang.cos(), ang.sin())[None, :, None, :]
    i = torch.arange(S, device=tok.device)
    see = (i[None, :] <= i[:, None]) & ((i[:, None] - i[None, :] < cfg.window) | (i[None, :] < cfg.sinks))

    def norm(x, w):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + cfg.eps) * w

    def rope(x):
        c = torch.complex(x[..., : d // 2], x[..., d // 2:]) * turn
        return torch.cat([c.real, c.imag], -1)

    x = W["embed.tok"][tok]
    for n in range(cfg.layers):
        p = lambda name: W[f"layer{n}.{name}"]
        qkv = (norm(x, p("attn_norm")) @ p("wqkv").t()).view(B, S, nh + 2 * nkv, d)
        q, k, v = rope(norm(qkv[:, :, :nh], p("q_norm"))), rope(norm(qkv[:, :, nh:nh + nkv], p("k_norm"))), qkv[:, :, nh + nkv:]
        k, v = (t.repeat_interleave(nh // nkv, 2) for t in (k, v))
        s = torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(d)
        a = torch.einsum("bhij,bjhd->bihd", torch.softmax(s.masked_fill(~see, -math.inf), -1), v)
        x = x + a.reshape(B, S, nh * d) @ p("wo").t()
        gu = norm(x, p("mlp_norm")) @ p("w13").t()
        x = x + (torch.nn.functional.silu(gu[..., : cfg.ffn]) * gu[..., cfg.ffn:]) @ p("w2").t()
    z = norm(x, W["head.norm"]) @ W["head.out"].t()
    ce = -torch.log_softmax(z, -1).gather(-1, tgt[..., None])[..., 0]
    t = distill.temperature
    logp, logq = torch.log_softmax(values.to(dtype) / t, -1), torch.log_softmax(z / t, -1).gather(-1, ids.long())
    loss = ((1 - distill.weight) * ce + distill.weight * t * t * (logp.exp() * (logp - logq)).sum(-1)).mean()
    loss.backward()
    return float(loss.detach()), {k: v.grad for k, v in W.items()}


@pytest.mark.parametrize("heads, kv, hidden", [(4, 2, 256), (2, 1, 256)])
def test_first_update_follows_the_gradient(heads, kv, hidden):
    """As for the plain decoder: with zero moments the first update has the sign of the gradient, parameter by parameter."""
    from rocm_systems_b200.models.llama import DistillConfig, LlamaConfig, LlamaTrainer
    from rocm_systems_b200.parallel.fsdp import AdamWConfig

    cfg = LlamaConfig(vocab=1024, hidden=hidden, layers=2, heads=heads, kv_heads=kv, ffn=512, seq_len=200, qk_norm=True, window=50, sinks=3)
    distill = DistillConfig(weight=0.6, temperature=2.0)
    dev = torch.device("cuda", 0)
    tr = LlamaTrainer(cfg, None, dev, opt=AdamWConfig(lr=1e-3, weight_decay=0.0), seed=5, distill=distill)
    g = torch.Generator().manual_seed(3)
    tok, tgt = (torch.randint(0, cfg.vocab, (2, cfg.seq_len), generator=g) for _ in range(2))
    ids = torch.stack([torch.randperm(cfg.vocab, generator=g)[:9] for _ in range(2 * cfg.seq_len)]).view(2, cfg.seq_len, 9)
    values = 2 * torch.randn(2, cfg.seq_len, 9, generator=g)
    units = [tr.embed, *tr.layers, tr.head]
    before = {f"{u.name}.{s.name}": u.master[u.offsets[s.name]:u.offsets[s.name] + s.numel].view(*s.shape).clone() for u in units for s in u.specs}
    assert sum(v.numel() for v in before.values()) == cfg.param_count()
    seen = {k: v.to(torch.bfloat16).float() for k, v in before.items()}
    ref_loss, grads = _reference(cfg, seen, tok.to(dev), tgt.to(dev), ids.to(dev), values.to(dev), distill)
    loss = tr.step(tok.pin_memory(), tgt.pin_memory(), teacher=(ids.pin_memory(), values.pin_memory()))
    assert abs(loss - ref_loss) < 0.02 * max(1.0, ref_loss), (loss, ref_loss)
    worst = []
    for u in units:
        for s in u.specs:
            name = f"{u.name}.{s.name}"
            o = u.offsets[s.name]
            delta = before[name] - u.master[o:o + s.numel].view(*s.shape)
            gr = grads[name].float()
            big = gr.abs() > 0.2 * gr.abs().max()
            agree = float((torch.sign(delta[big]) == torch.sign(gr[big])).float().mean())
            worst.append((agree, float((delta[big].abs() > 0.5e-3).float().mean()), name))
    assert all(a >= 0.98 and m >= 0.98 for a, m, _ in worst), worst
    from rocm_systems_b200.ops import train_ops

    assert train_ops.gemm_take_error() == 0


def test_eval_runs_the_same_layers_and_a_teacher_needs_its_configuration():
    from rocm_systems_b200.models.llama import LlamaConfig, LlamaTrainer

    cfg = LlamaConfig(vocab=1024, hidden=256, layers=2, heads=4, kv_heads=2, ffn=512, seq_len=64, qk_norm=True, window=20, sinks=1)
    tr = LlamaTrainer(cfg, None, torch.device("cuda", 0), seed=7)
    g = torch.Generator().manual_seed(11)
    tok, tgt = (torch.randint(0, cfg.vocab, (2, cfg.seq_len), generator=g) for _ in range(2))
    l_eval = tr.eval_loss(tok, tgt)
    assert abs(tr.step(tok, tgt) - l_eval) < 0.05
    with pytest.raises(AssertionError, match="DistillConfig"):
        tr.step(tok, tgt, teacher=(torch.zeros(2, 64, 3, dtype=torch.int64), torch.zeros(2, 64, 3)))


def test_tensor_parallel_attention_with_a_window():
    """One rank's attention half with a window against the plain formula, forward and backward."""
    from rocm_systems_b200.comm import Communicator, get_unique_id
    from rocm_systems_b200.parallel.tp import TensorParallelAttention

    torch.cuda.set_device(0)
    comm = Communicator(0, 1, get_unique_id(), 0)
    rows, hidden, heads, kv, seq = 512, 512, 8, 4, 256
    layer = TensorParallelAttention(comm, rows, hidden, heads, kv, seq, seed=3, window=60, sinks=2)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = ((s * torch.randn(rows, hidden, device="cuda", generator=g)).to(torch.bfloat16) for s in (1.0, 0.1))
    y, dx = layer.forward(x).clone(), layer.backward(dy).clone()
    d = hidden // heads
    xf, wq, wo = (t.double().requires_grad_(True) for t in (x, layer.w_qkv, layer.w_o))
    qkv = (xf @ wq.t()).view(rows // seq, seq, heads + 2 * kv, d)
    turn = torch.complex(layer.rope[..., 0].double(), layer.rope[..., 1].double())[None, :, None, :]

    def rope(t):
        c = torch.complex(t[..., : d // 2], t[..., d // 2:]) * turn
        return torch.cat([c.real, c.imag], -1)

    q, k, v = rope(qkv[:, :, :heads]), rope(qkv[:, :, heads:heads + kv]), qkv[:, :, heads + kv:]
    k, v = (t.repeat_interleave(heads // kv, 2) for t in (k, v))
    i = torch.arange(seq, device="cuda")
    see = (i[None, :] <= i[:, None]) & ((i[:, None] - i[None, :] < 60) | (i[None, :] < 2))
    p = torch.softmax((torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(d)).masked_fill(~see, -math.inf), -1)
    ref = torch.einsum("bhij,bjhd->bihd", p, v).reshape(rows, hidden) @ wo.t()
    grads = torch.autograd.grad(ref, (xf, wq, wo), dy.double())
    # five roundings to bf16 one after another, each at most 2^-8 of its value: in the 2-norm below 5 * 2^-8
    for got, want in ((y, ref), (dx, grads[0]), (layer.grads["w_qkv"], grads[1]), (layer.grads["w_o"], grads[2])):
        assert float((got.double() - want).norm() / want.norm()) < 5 * 2.0 ** -8
    layer.free()
    comm.destroy()
