"""The C entry points and Python modules of the embedding, the products with an
epilogue and the gradient clip: their argument checks, before anything touches a device."""
from array import array

import pytest
import torch

from mimansm1_v1_amd import _lib, embedding, grad_clip

FAKE = 1 << 20   # aligned, non-null, never dereferenced


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def lookup(lib, ids=FAKE, wide=1, w=FAKE, w32=1, ldw=64, out=FAKE, o32=0, ldo=64, n=10, vocab=100, dim=64):
    return lib.mm1_embedding(ids, wide, w, w32, ldw, out, o32, ldo, 1.0, n, vocab, dim, None)


def test_lookup_argument_errors(lib):
    for kw in (dict(ids=None), dict(w=None), dict(out=None)):
        assert lookup(lib, **kw) == -1
    for kw in (dict(n=-1), dict(vocab=0), dict(dim=0), dict(ldw=63), dict(ldo=63), dict(n=(1 << 26) + 1),
               dict(vocab=(1 << 30) + 1), dict(n=1 << 26, dim=1024, ldw=1024, ldo=1024)):
        assert lookup(lib, **kw) == -2, kw
    for kw in (dict(ids=FAKE + 4), dict(ids=FAKE + 2, wide=0), dict(w=FAKE + 2), dict(out=FAKE + 1)):
        assert lookup(lib, **kw) == -6, kw
    assert lookup(lib, n=0, ids=None, out=None) == 0


def grad(lib, ids=FAKE, wide=1, dy=FAKE, ld_dy=64, g=FAKE, g32=1, ldg=64, padding=-1, acc=0, ws=FAKE, nb=None, n=100,
         vocab=100, dim=64):
    nb = lib.mm1_embedding_grad_workspace_size(n, vocab, dim) if nb is None else nb
    return lib.mm1_embedding_grad(ids, wide, dy, 0, ld_dy, g, g32, ldg, 1.0, padding, acc, ws, nb, n, vocab, dim, None)


def test_gradient_argument_errors(lib):
    for kw in (dict(ids=None), dict(dy=None), dict(g=None)):
        assert grad(lib, **kw) == -1
    for kw in (dict(n=-1), dict(ld_dy=63), dict(ld_dy=-64), dict(ldg=63), dict(padding=-2), dict(padding=100),
               dict(dim=0)):
        assert grad(lib, **kw) == -2, kw
    need = lib.mm1_embedding_grad_workspace_size(100, 100, 64)
    assert grad(lib, nb=need - 1) == -4 and grad(lib, ws=None) == -4
    for kw in (dict(ids=FAKE + 4), dict(dy=FAKE + 1), dict(g=FAKE + 2), dict(ws=FAKE + 8)):
        assert grad(lib, **kw) == -6, kw
    assert grad(lib, n=0, acc=1, ids=None, dy=None) == 0


def test_gradient_workspace_sizes(lib):
    """Sorted (id, token) pairs of 8 bytes; beyond 16384 tokens a second copy and
    the digit counts of each tile of 8192 and pass; beyond a unit of tokens (8,
    16 from 8193 on, 32 from 16385 on, 48 from 32769 on) two fp32 rows per unit.  Regions start at multiples of 256 bytes."""
    up = lambda x: (x + 255) // 256 * 256
    size = lib.mm1_embedding_grad_workspace_size
    assert size(0, 100, 64) == 0
    assert size(7, 100, 64) == up(8 * 7)
    assert size(100, 100, 64) == up(800) + up(13 * 2 * 64 * 4)
    n = 20000
    assert size(n, 49152, 1280) == 2 * up(8 * n) + up(2 * 256 * 3 * 4) + up(625 * 2 * 1280 * 4)
    assert size(-1, 100, 64) == 0 and size(10, 0, 64) == 0


def clip(lib, count=2, ptrs=(FAKE, FAKE + 4096), out=None, rows=None, cols=(10, 20), ld=None, ld_out=None, f32=(1, 0),
         norm_type=0, max_norm=1.0, eps=1e-6, norm=FAKE, ws=FAKE, nb=None, scale=True):
    at = lambda kind, v: None if v is None else array(kind, v)
    keep = [at("Q", ptrs), at("l", rows), at("l", cols), at("l", ld), at("Q", out), at("l", ld_out)]
    p, r, c, l, o, lo = (None if a is None else a.buffer_info()[0] for a in keep)
    nb = lib.mm1_grad_norm_workspace_size(max(count, 0)) if nb is None else nb
    f32 = None if f32 is None else bytes(f32)
    if not scale:
        return lib.mm1_grad_norm(count, p, r, c, l, f32, norm_type, norm, ws, nb, None)
    return lib.mm1_grad_clip(count, p, o, r, c, l, lo, f32, norm_type, max_norm, eps, 0, norm, ws, nb, None)


@pytest.mark.parametrize("scale", [False, True])
def test_clip_argument_errors(lib, scale):
    for kw in (dict(norm=None), dict(ptrs=None), dict(cols=None), dict(f32=None), dict(ptrs=(FAKE, 0)),
               dict(rows=(1, 1), ld=None)):
        assert clip(lib, scale=scale, **kw) == -1, kw
    for kw in (dict(count=-1), dict(cols=(-1, 2)), dict(norm_type=2), dict(rows=(1, -1), ld=(10, 20), ld_out=(10, 20)),
               dict(rows=(2, 2), ld=(9, 20), ld_out=(10, 20)), dict(cols=(1 << 41, 2)),
               dict(rows=((1 << 31) - 1, 1), ld=(10, 20), ld_out=(10, 20))):
        assert clip(lib, scale=scale, **kw) == -2, kw
    assert clip(lib, scale=scale, ws=None) == -4 and clip(lib, scale=scale, nb=100) == -4
    for kw in (dict(ptrs=(FAKE + 2, FAKE)), dict(ptrs=(FAKE, FAKE + 1)), dict(norm=FAKE + 2), dict(ws=FAKE + 8)):
        assert clip(lib, scale=scale, **kw) == -6, kw


def test_clip_only_argument_errors(lib):
    for kw in (dict(out=(FAKE, 0)), dict(rows=(1, 1), ld=(10, 20), out=(FAKE, FAKE))):
        assert clip(lib, **kw) == -1, kw
    for kw in (dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(eps=-1.0), dict(eps=float("inf")),
               dict(out=(FAKE, FAKE), rows=(2, 2), ld=(10, 20), ld_out=(9, 20))):
        assert clip(lib, **kw) == -2, kw
    assert clip(lib, out=(FAKE + 2, FAKE)) == -6


def test_modules_refuse_cpu_tensors():
    w, ids, g = torch.zeros(10, 8), torch.zeros(4, dtype=torch.int64), torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        embedding.embed(ids, w)
    with pytest.raises(ValueError, match="CUDA"):
        embedding.embedding_grad(ids, g, 10)
    with pytest.raises(TypeError):
        embedding.embed([1, 2], w)
    with pytest.raises(ValueError, match="CUDA"):
        grad_clip.grad_norm([g])
    with pytest.raises(ValueError, match="norm_type"):
        grad_clip.grad_norm([g], 1.0)


@pytest.mark.parametrize("make,want", [
    (lambda b: b, (1, 120, 120)), (lambda b: b.t(), (1, 120, 120)), (lambda b: b[:, 2:7], (10, 5, 12)),
    (lambda b: b[:, 2:7].t(), (10, 5, 12)), (lambda b: b[3:5], (1, 24, 24)), (lambda b: b[2, 3], (1, 1, 1)),
    (lambda b: b[:, :1], (10, 1, 12)), (lambda b: b[:, ::2], (60, 1, 2)), (lambda b: b[:, ::5], None), (lambda b: b[:1].expand(4, 12), None),
    (lambda b: b.view(2, 5, 12)[:, :3], (2, 36, 60)), (lambda b: b.view(10, 3, 4)[:, :2, :3], None)])
def test_runs_of_strided_tensors(make, want):
    """Rows of consecutive values: (rows, cols, distance), None for what is not."""
    t = make(torch.arange(120.).view(10, 12))
    runs = grad_clip._runs(t)
    assert (runs if want is None else runs[1:]) == want


def product(lib, x=FAKE, xl=0, ldx=256, w=FAKE, wl=0, ldw=256, bias=None, bias32=1, act=0, res=None, res32=0, ldr=64,
            pre=None, ldp=64, out=FAKE, out32=0, ldo=64, ws=FAKE, nb=1 << 30, m=100, n=64, k=256):
    return lib.mm1_linear(x, xl, ldx, w, wl, ldw, bias, bias32, act, res, res32, ldr, pre, ldp, out, out32, ldo, ws,
                          nb, m, n, k, None)


def test_linear_argument_errors(lib):
    for kw in (dict(x=None), dict(w=None), dict(out=None)):
        assert product(lib, **kw) == -1
    for kw in (dict(m=0), dict(n=0), dict(k=0), dict(k=257), dict(xl=2), dict(wl=-1), dict(xl=1, wl=0), dict(ldx=255),
               dict(ldx=250), dict(ldw=248), dict(ldw=260), dict(wl=1, ldw=56), dict(wl=1, n=57, ldw=56),
               dict(xl=1, wl=1, ldx=96, ldw=64), dict(xl=1, wl=1, ldx=104, ldw=64, act=1), dict(act=5), dict(act=-1),
               dict(ldo=63), dict(ldo=(1 << 24) + 1), dict(res=FAKE, ldr=63), dict(act=4, pre=FAKE, ldp=63),
               dict(pre=FAKE), dict(ldx=1 << 23), dict(m=(1 << 28) + 1)):
        assert product(lib, **kw) == -2, kw
    for kw in (dict(x=FAKE + 8), dict(w=FAKE + 8), dict(ws=FAKE + 8), dict(out=FAKE + 1), dict(out=FAKE + 2, out32=1),
               dict(bias=FAKE + 2), dict(res=FAKE + 1), dict(act=4, pre=FAKE + 1)):
        assert product(lib, **kw) == -6, kw
    size = lib.mm1_linear_workspace_size
    need = size(64, 64, 4096, 0, 0, 0)
    assert need > 0 and size(0, 64, 64, 0, 0, 0) == 0 and size(64, 64, 4096, 1, 0, 0) == 0
    assert size(16, 64, 4096, 0, 0, 0) == size(16, 64, 4096, 0, 1, 0) == 0      # one launch for a few rows
    assert size(16, 64, 8192, 0, 0, 0) > 0 and size(16, 64, 8192, 0, 1, 0) > 0      # ... not for sums this long
    assert product(lib, m=64, k=4096, ldx=4096, ldw=4096, nb=need - 1) == -4
    assert product(lib, m=64, k=4096, ldx=4096, ldw=4096, ws=None) == -4


def test_linear_refuses_strides_past_its_offsets(lib):
    """A wave's 128 rows of the output or residual, or M where that is fewer, have
    32-bit byte offsets: (rows - 1) ld + 64 elements at most 2^32 bytes.  What the
    sizes let through is refused for its address, so that nothing is launched."""
    far = ((1 << 30) - 64) // 127
    for kw in (dict(m=1000, ldo=far + 1, out32=1), dict(m=128, ldo=1 << 24, out32=1),
               dict(m=1000, res=FAKE, res32=1, ldr=far + 1), dict(m=64, ldo=(1 << 24) + 1),
               dict(m=66, res=FAKE, res32=1, ldr=1 << 24)):
        assert product(lib, **kw) == -2, kw
    for kw in (dict(m=1000, ldo=far, out32=1), dict(m=64, ldo=1 << 24, out32=1), dict(m=1000, ldo=1 << 24),
               dict(m=1000, res=FAKE, ldr=1 << 24), dict(m=1000, res=FAKE, res32=1, ldr=1 << 23),
               dict(m=1000, act=4, pre=FAKE, ldp=1 << 24)):
        assert product(lib, x=FAKE + 8, **kw) == -6, kw
    wide = 8 * (far // 8 + 1)        # dX's and dW's rows are theirs whole
    kw = dict(m=200, n=200, ldy=200, ldp=200, ldx=wide, ldw=wide, k=wide, db=None)
    assert backward(lib, dx32=1, dw=None, **kw) == -2 and backward(lib, dx=None, dw32=1, **kw) == -2
    assert backward(lib, dx32=1, dw=None, dy=FAKE + 1, **dict(kw, m=16)) == -6
    assert backward(lib, dy=FAKE + 1, **kw) == -6


def backward(lib, dy=FAKE, dy32=0, ldy=60, pre=FAKE, ldp=60, act=4, x=FAKE, ldx=40, w=FAKE, wl=0, ldw=40, dx=FAKE, dx32=0,
             dw=FAKE, dw32=0, db=FAKE, db32=1, ws=FAKE, nb=None, m=100, n=60, k=40):
    nb = lib.mm1_linear_backward_workspace_size(m, n, k, 1, 1, 1, 1) if nb is None else nb
    return lib.mm1_linear_backward(dy, dy32, ldy, pre, ldp, act, x, ldx, w, wl, ldw, dx, dx32, dw, dw32, db, db32, ws, nb,
                                   m, n, k, None)


def test_linear_backward_argument_errors(lib):
    for kw in (dict(dy=None), dict(pre=None), dict(dx=None, dw=None, db=None), dict(x=None), dict(w=None)):
        assert backward(lib, **kw) == -1, kw
    for kw in (dict(m=0), dict(n=0), dict(n=(1 << 24) + 1), dict(act=5), dict(act=-1), dict(ldy=59), dict(ldp=59),
               dict(ldx=32), dict(ldx=44), dict(ldw=32), dict(wl=1, ldw=56), dict(wl=2), dict(k=41)):
        assert backward(lib, **kw) == -2, kw
    size = lib.mm1_linear_backward_workspace_size
    need = size(100, 60, 40, 1, 1, 1, 1)
    assert need >= 100 * 64 * 2 + 7 * 60 * 4          # dz at 64 columns; partial sums of 7 blocks of 16 rows
    assert size(100, 60, 40, 0, 0, 0, 1) == size(100, 60, 40, 1, 0, 0, 1) == 7 * 60 * 4
    assert size(100, 64, 40, 0, 1, 0, 0) == 0 and size(0, 64, 40, 1, 1, 1, 1) == 0
    assert backward(lib, nb=need - 1) == -4 and backward(lib, ws=None) == -4
    for kw in (dict(dy=FAKE + 1), dict(pre=FAKE + 1), dict(x=FAKE + 8), dict(w=FAKE + 8), dict(dx=FAKE + 1),
               dict(dw=FAKE + 2, dw32=1), dict(db=FAKE + 2), dict(ws=FAKE + 8)):
        assert backward(lib, **kw) == -6, kw


def test_pack_argument_errors(lib):
    pack = lambda src=FAKE, f32=1, ld=30, rows=10, cols=30, dst=FAKE, ldd=32, out=16: \
        lib.mm1_pack_bf16(src, f32, ld, rows, cols, dst, ldd, out, None)
    assert pack(src=None) == -1 and pack(dst=None) == -1
    for kw in (dict(rows=0), dict(cols=0), dict(out=9), dict(ld=29), dict(ldd=30), dict(ldd=24)):
        assert pack(**kw) == -2, kw
    assert pack(src=FAKE + 2) == -6 and pack(dst=FAKE + 8) == -6


def test_linear_refuses_cpu_tensors():
    from mimansm1_v1_amd import linear
    with pytest.raises(ValueError, match="CUDA"):
        linear.fused_linear(torch.zeros(2, 8), torch.zeros(4, 8))
    with pytest.raises(TypeError):
        linear.fused_linear([1.0], torch.zeros(4, 8))


def test_linear_refuses_sizes_past_the_librarys():
    """The documented widths, which an operand's own checks let past for one of the
    two, and row counts before they wrap in a 32-bit argument."""
    from mimansm1_v1_amd import linear
    check = linear._check_sizes
    check(1 << 28, 4_000_000, 1)
    check(0, 1, 4_000_000)
    for rows, n, k in ((1, 4_000_001, 8), (1, 8, 4_000_001), (1, (1 << 32) + 8, 8), ((1 << 28) + 1, 8, 8),
                       ((1 << 32) + 5, 8, 8)):
        with pytest.raises(ValueError, match="at most"):
            check(rows, n, k)


def test_embedding_refuses_sizes_past_the_librarys():
    """Rows and columns before they wrap in a 32-bit argument."""
    check = embedding._check_sizes
    check(1 << 30, 1)
    check(1, (1 << 31) - 1)
    for vocab, dim in ((0, 8), (8, 0), ((1 << 30) + 1, 8), ((1 << 32) + 10, 8), (8, (1 << 32) + 8)):
        with pytest.raises(ValueError, match="rows are taken"):
            check(vocab, dim)


@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_tangents_are_refused(grad_mode):
    """No call drops a tangent: each raises before it looks at devices."""
    from torch.autograd import forward_ad

    from mimansm1_v1_amd import linear, swiglu
    ids = torch.zeros(4, dtype=torch.int64)
    square = lambda: torch.zeros(4, 4)
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        dual = forward_ad.make_dual(square(), torch.ones(4, 4))
        row = forward_ad.make_dual(torch.zeros(4), torch.ones(4))
        calls = [lambda: linear.fused_linear(dual, square()), lambda: linear.fused_linear(square(), dual),
                 lambda: linear.fused_linear(square(), square(), row),
                 lambda: linear.fused_linear(square(), square(), residual=dual),
                 lambda: linear.Linear(4, 4)(dual), lambda: embedding.embed(ids, dual),
                 lambda: embedding.embedding_grad(ids, dual, 4),
                 lambda: embedding.embedding_grad(ids, square(), 4, out=dual),
                 lambda: grad_clip.grad_norm([square(), dual]), lambda: grad_clip.clip_grads([dual], 1.0),
                 lambda: grad_clip.clip_grads([square()], 1.0, out=[dual])]
        calls += [lambda i=i: swiglu.fused_swiglu(*(dual if j == i else square() for j in range(4)), residual=square())
                  for i in range(4)]
        calls.append(lambda: swiglu.fused_swiglu(*(square() for _ in range(4)), residual=dual))
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        parameter = torch.nn.Parameter(square())
        parameter.grad = dual
        with pytest.raises(NotImplementedError, match="forward-mode"):
            grad_clip.clip_grad_norm_([parameter], 1.0)
        # beside duals that are not an input's, calls go on as ever
        with pytest.raises(ValueError, match="CUDA"):
            linear.fused_linear(square(), square())


def test_memory_shared_with_the_gradients_output():
    """Shared values are found whatever the views; neighbours, other columns of the
    same rows and other rows are let through."""
    store = torch.zeros(40, 16)
    out = store[:10, :8]
    for t in (out, store[:4, :8], store[9:12, :8], store[2:6, 7:9], store[::3, 4:10], store.view(-1)[:80].view(10, 8),
              store[:10, :8].t(), store[0, 3], store[:5, 12:].as_strided((5, 8), (16, 1)), store[3].expand(4, 16),
              store.view(20, 2, 16)[:, :, :2], store.view(torch.int32)[5], store.view(torch.int64)[:, 3:5],
              store.view(-1)[-632:].view(79, 8), store[:, 7], store.view(torch.int64)[:, 0]):
        assert embedding._shares(out, t), (t.shape, t.stride())
    for t in (store[10:20, :8], store[:10, 8:], store[::2, 9:12], torch.zeros(10, 8), store[:0, :8], store[12, 8:].expand(4, 8),
              store.view(torch.int64)[:, 4:], store.view(2, 20, 16)[:, ::5, 10:], store[0, 8:], store[20:30, :8],
              store[:, 9], store.view(torch.int64)[:, 7], store[2, 12], store[:0]):
        assert not embedding._shares(out, t), (t.shape, t.stride())
    assert embedding._shares(store, store[3:4, 2:3]) and not embedding._shares(store[:10], store[10:])
    assert embedding._shares(store[3:4], store[3]) and not embedding._shares(store[3:4], store[4])


def test_swiglu_refuses_other_output_types():
    from mimansm1_v1_amd import swiglu
    ts = [torch.zeros(128, 128, dtype=torch.bfloat16)] * 4
    for residual in (None, ts[0]):
        for bad in (torch.float16, torch.float64, "fp32"):
            with pytest.raises(TypeError, match="out_dtype"):
                swiglu.fused_swiglu(*ts, residual, bad)


def test_clip_outputs_in_a_gradient_given_twice():
    """A gradient that is given twice is read twice, so an output may lie in neither's
    memory, whichever of the two it belongs to."""
    a, b, c = (torch.zeros(6, 4) for _ in range(3))
    refuse = grad_clip._Table._refuse_shared
    for out in ([a, b], [b, a], [a, a]):
        with pytest.raises(ValueError, match="memory of gradient"):
            refuse([a, a], out)
    with pytest.raises(ValueError, match="memory of gradient 0"):
        refuse([a, b, a], [c, b, a])
    refuse([a, b], [a, c])
    refuse([a, a, b], [torch.zeros(6, 4), c, b])
