"""The operators of a training step as they are used together: token ids through
the embedding, an attention and a feed-forward sublayer whose outputs join the
residual stream in their last product's epilogue, the tied head's loss, the
backward, and the clip of all gradients -- against the same step on torch's
embedding, additions and clip around the same sublayers, and against
differences of the loss."""
import pytest
import torch
import torch.nn as nn

import mimansm1_v1_amd as mm
from mimansm1_v1_amd import attention as A
from mimansm1_v1_amd import lm_head as L
from mimansm1_v1_amd import swiglu as S

pytestmark = pytest.mark.gpu

D, VOCAB, SEQ = 256, 512, 96


class Model(nn.Module):
    """Two blocks of width 256 around the package's sublayers; fused: on the
    step's operators, else torch's in their place."""

    def __init__(self, fused, stream, seed=0):
        super().__init__()
        torch.manual_seed(seed)
        self.fused, self.stream = fused, stream
        cfg = A.AttnConfig(d_model=D, n_heads=2, n_kv_heads=1, max_seq_len=SEQ)
        rope = A.Rotary(cfg.head_dim, SEQ, cfg.rope_theta)
        weight = torch.randn(VOCAB, D)
        self.embedding = mm.Embedding(VOCAB, D, scale=0.5, out_dtype=stream) if fused else nn.Embedding(VOCAB, D)
        self.embedding.weight.data.copy_(weight)
        self.blocks = nn.ModuleList(nn.ModuleList([A.Attention(cfg, rope), S.SwiGLU(S.FFNConfig(D, 384))])
                                    for _ in range(2))
        self.head = L.LMHead(L.HeadConfig(d_model=D, vocab=VOCAB), self.embedding)

    def forward(self, ids, targets):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            h = self.embedding(ids) if self.fused else (self.embedding(ids) * 0.5).to(self.stream)
            for attn, ffn in self.blocks:
                h = attn(h, residual=h) if self.fused else h + attn(h)
                h = ffn(h, residual=h) if self.fused else h + ffn(h)
            return self.head(h, targets)


def batch(dev, seed=1):
    g = torch.Generator(dev).manual_seed(seed)
    ids = torch.randint(0, VOCAB, (3, SEQ), device=dev, generator=g)
    targets = torch.roll(ids, -1, 1)
    targets[:, -1] = L.IGNORE_INDEX
    return ids, targets


@pytest.mark.parametrize("stream", [torch.float32, torch.bfloat16])
def test_step_matches_torch_around_the_same_sublayers(hip_device, stream):
    """Loss, every gradient, the norm and the clipped gradients.  The two differ
    by where the sublayers' outputs are rounded: to bf16 before the addition in
    torch's step (h = 2^-8 of them, twice a block), once after it here."""
    ids, targets = batch(hip_device)
    got = []
    for fused in (True, False):
        model = Model(fused, stream).to(hip_device)
        loss = model(ids, targets)
        loss.backward()
        grads = {n: p.grad.clone() for n, p in model.named_parameters()}
        assert all(bool(torch.isfinite(g).all()) for g in grads.values())
        clip = mm.clip_grad_norm_ if fused else nn.utils.clip_grad_norm_
        norm = clip(model.parameters(), 0.1)
        got.append((loss.detach(), grads, norm, {n: p.grad for n, p in model.named_parameters()}))
    (loss, grads, norm, clipped), (loss0, grads0, norm0, clipped0) = got
    assert (loss - loss0).abs() <= 2e-2 * loss0.abs()
    # four additions, each within 2 h of a stream that they dominate, through slopes of order one
    for n in grads0:
        off = (grads[n] - grads0[n]).norm() / grads0[n].norm()
        assert off <= 4 * 2 * 2.0 ** -8, (n, off.item())
    assert (norm - norm0).abs() <= 4 * 2 * 2.0 ** -8 * norm0 and norm > 0.1
    total = mm.grad_norm([clipped[n] for n in clipped])
    assert abs(total.item() - 0.1) <= 0.1 * (1e-5 + 8 * 2.0 ** -24)
    want = 0.1 / (norm.item() + 1e-6)
    for n in grads:
        assert bool(((clipped[n] - grads[n] * want).abs() <= 8 * 2.0 ** -24 * want * grads[n].abs() + 1e-30).all())


def test_residual_equals_addition(hip_device):
    """forward(x, residual=r) against r + forward(x) for each sublayer, dtype and
    backend: equal but for the one rounding that it saves (half a step of bf16 of
    the sublayer's output, and of the sum in a bf16 stream)."""
    torch.manual_seed(0)
    cfg = A.AttnConfig(d_model=D, n_heads=2, n_kv_heads=1, max_seq_len=SEQ)
    attn = A.Attention(cfg, A.Rotary(cfg.head_dim, SEQ, cfg.rope_theta)).to(hip_device)
    ffn = S.SwiGLU(S.FFNConfig(D, 384)).to(hip_device)
    h = 2.0 ** -8
    for module in (attn, ffn):
        for backend in ("hip", "math"):
            for x_type in (torch.float32, torch.bfloat16):
                for r_type in (torch.float32, torch.bfloat16, torch.float64):
                    x = torch.randn(2, SEQ, D, device=hip_device).to(x_type)
                    r = torch.randn(2, SEQ, D, device=hip_device).to(r_type)
                    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
                        y, got = module(x, backend), module(x, backend, residual=r)
                    want = r + y
                    assert got.dtype == want.dtype
                    bound = h * y.abs().double() + (2 * h * want.abs().double() if got.dtype == torch.bfloat16 else 0)
                    bound = bound + 2.0 ** -12 * y.abs().max()      # sums in another order, before the rounding
                    assert bool(((got.double() - want.double()).abs() <= bound).all())
        with pytest.raises(ValueError, match="residual"):
            module(x, residual=r[:, 1:])


def test_gradient_against_differences(hip_device):
    """The loss's slope along one direction of the embedding and of a down
    projection, from central differences of the loss itself; the loss's
    rounding to bf16 products bounds how near they can be."""
    ids, targets = batch(hip_device)
    model = Model(True, torch.float32).to(hip_device)
    loss = model(ids, targets)
    loss.backward()
    for p in (model.embedding.weight, model.blocks[0][1].w_down):
        v = p.grad / p.grad.norm()
        slope = (p.grad * v).sum().item()
        keep, side = p.data.clone(), []
        step = 0.25 / max(slope, 1.0)
        for s in (1, -1):
            p.data.copy_(keep + s * step * v)
            with torch.no_grad():
                side.append(model(ids, targets).item())
        p.data.copy_(keep)
        measured = (side[0] - side[1]) / (2 * step)
        # 5%: two losses each within 2^-8 of 6 over a difference of 2 step slope
        assert abs(measured - slope) <= 0.05 * slope + 2 * 2.0 ** -8 * loss.item() / (2 * step), (measured, slope)


def test_two_steps_repeat_bitwise(hip_device):
    """The embedding's and the products' sums have a fixed order: a step's
    gradients repeat."""
    ids, targets = batch(hip_device)
    runs = []
    for _ in range(2):
        model = Model(True, torch.float32).to(hip_device)
        model(ids, targets).backward()
        mm.clip_grad_norm_(model.parameters(), 0.1)
        runs.append([p.grad for p in model.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_greedy_single_tokens_without_gradients(hip_device):
    """The lookup and the products' epilogue for single tokens under no_grad:
    equal to the same rows of a longer batch's, whose tiles differ, within the
    sums' order."""
    torch.manual_seed(3)
    emb = mm.Embedding(VOCAB, D, out_dtype=torch.bfloat16, device=hip_device)
    ids = torch.randint(0, VOCAB, (200,), device=hip_device)
    w = (torch.randn(D, D, device=hip_device) / 16).to(torch.bfloat16)
    with torch.no_grad():
        x = emb(ids)
        assert torch.equal(emb(ids[:1]), x[:1])
        full = mm.fused_linear(x, w, residual=x, out_dtype=torch.float32)
        for i in (0, 77, 199):
            one = mm.fused_linear(x[i], w, residual=x[i], out_dtype=torch.float32)
            size = x[i].float().abs() @ w.float().abs().t() + x[i].float().abs()
            assert one.shape == (D,) and bool(((one - full[i]).abs() <= 2 * (D + 2) * 2.0 ** -24 * size).all())


@pytest.mark.parametrize("train", [False, True])
def test_swiglu_output_type_without_a_residual(hip_device, train):
    """fused_swiglu(..., out_dtype): fp32 outputs are the same sums before their one
    rounding, so that rounding them gives the bf16 ones but for the sums' order;
    gradients flow through both."""
    gen = torch.Generator(hip_device).manual_seed(5)
    randn = lambda *s: torch.randn(*s, device=hip_device, generator=gen).to(torch.bfloat16)
    x, ws = randn(70, D), [randn(D, 384) / 16, randn(D, 384) / 16, randn(384, D) / 16]
    leaves = [t.requires_grad_(train) for t in (x, *ws)]
    wide, half = S.fused_swiglu(*leaves, out_dtype=torch.float32), S.fused_swiglu(*leaves)
    assert wide.dtype == torch.float32 and half.dtype == torch.bfloat16
    assert torch.equal(S.fused_swiglu(*leaves, out_dtype=torch.bfloat16), half)
    with torch.no_grad():
        act = S.fused_swiglu(x, ws[0], ws[1], torch.eye(384, device=hip_device, dtype=torch.bfloat16))
    size = act.double().abs() @ ws[2].detach().double().abs()
    want = act.double() @ ws[2].detach().double()
    bound = 384 * 2.0 ** -24 * size                  # of 384 fp32 additions
    assert bool(((wide.detach().double() - want).abs() <= 1.01 * bound + 2.0 ** -24 * want.abs()).all())
    assert bool(((half.detach().double() - want).abs() <= 1.01 * bound + 2.0 ** -8 * (want.abs() + bound)).all())
    if train:
        dy = randn(70, D)
        for a, b in zip(torch.autograd.grad(wide, leaves, dy.float()), torch.autograd.grad(half, leaves, dy)):
            # the same bf16 products, summed in other orders and rounded to bf16 at each of two steps
            assert (a.double() - b.double()).norm() <= 4 * 2.0 ** -8 * b.double().norm()


@pytest.mark.parametrize("x_type", [torch.float16, torch.float64])
def test_residual_beside_inputs_of_other_types(hip_device, x_type):
    """Inputs that the sublayer takes without a residual it takes with one, in the
    addition's type."""
    torch.manual_seed(0)
    ffn = S.SwiGLU(S.FFNConfig(D, 384)).to(hip_device)
    x = torch.randn(2, SEQ, D, device=hip_device).to(x_type)
    for r_type in (torch.float32, torch.bfloat16):
        r = torch.randn(2, SEQ, D, device=hip_device).to(r_type)
        with torch.no_grad():
            y, got = ffn(x), ffn(x, residual=r)
        want = r + y
        assert got.dtype == want.dtype
        # y is rounded to bf16 before the addition there, and the sums' order differs
        bound = 2.0 ** -8 * y.double().abs() + 2.0 ** -12 * y.double().abs().max() + 2.0 ** -24 * want.double().abs()
        assert bool(((got.double() - want.double()).abs() <= bound).all())
