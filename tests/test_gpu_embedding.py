"""The embedding lookup and its gradient (mimansm1_v1_amd/embedding.py) against
torch in the same arithmetic (lookup) and against 64-bit sums (gradient)."""
import math

import numpy as np
import pytest
import torch

from mimansm1_v1_amd import _lib, embedding, lm_head

pytestmark = pytest.mark.gpu

FP32, BF16 = torch.float32, torch.bfloat16


def make_ids(kind, n, vocab, gen, dev, dtype=torch.int64):
    ids = torch.randint(0, vocab, (n,), generator=gen, device=dev)
    if kind == "same":
        ids.fill_(vocab - 1)
    elif kind == "few":
        ids = ids % 3
    elif kind == "outside":
        ids = torch.where(ids % 2 == 0, -100, vocab + ids)
    elif kind == "padded":
        ids[n - n // 4:] = -100
        ids[: n // 8] = vocab
    elif kind == "sorted":
        ids = ids.sort().values
    return ids.to(dtype)


def exact_grad(ids, dy, vocab, scale, skip=-1):
    """(sums, sums of magnitudes, tokens per row) in 64 bits, on the host."""
    ids, dy = ids.reshape(-1).long().cpu(), dy.reshape(-1, dy.shape[-1]).double().cpu()
    ok = (ids >= 0) & (ids < vocab) & (ids != skip)
    zero = torch.zeros(vocab, dy.shape[1], dtype=torch.float64)
    count = torch.bincount(ids[ok], minlength=vocab)
    return (zero.index_add(0, ids[ok], dy[ok]) * scale, zero.index_add(0, ids[ok], dy[ok].abs()) * abs(scale), count)


def check_grad(got, ids, dy, scale, old=None, skip=-1):
    """Within one rounding of each of the row's n fp32 additions, of the scale and
    of the addition to what was there, and of the result's type."""
    want, size, count = exact_grad(ids, dy, got.shape[0], scale, skip)
    if old is not None:
        want, size = want + old.double().cpu(), size + old.double().abs().cpu()
    u = 2.0 ** -24
    bound = (count[:, None] + 3) * u * 1.01 * size
    if got.dtype == BF16:
        bound = bound + torch.finfo(BF16).eps / 2 * (want.abs() + bound)
    worst = ((got.double().cpu() - want).abs() - bound).max().item()
    assert worst <= 0, worst
    if old is None:
        assert not got[(count == 0).to(got.device)].any()
    else:
        rest = (count == 0).to(got.device)
        assert torch.equal(got[rest], old[rest])


@pytest.mark.parametrize("n", [1, 7, 300])
@pytest.mark.parametrize("dim", [1, 7, 8, 649, 1280])
@pytest.mark.parametrize("w,o", [(FP32, BF16), (FP32, FP32), (BF16, BF16), (BF16, FP32)])
def test_lookup_equals_torch(hip_device, n, dim, w, o):
    gen = torch.Generator(hip_device).manual_seed(n * dim)
    weight = torch.randn(501, dim, device=hip_device, generator=gen).to(w)
    scale = math.sqrt(dim)
    for idtype in (torch.int64, torch.int32):
        ids = make_ids("padded", n, 501, gen, hip_device, idtype)
        ok = (ids >= 0) & (ids < 501)
        want = (weight[torch.where(ok, ids, 0)].float() * scale * ok[:, None]).to(o)
        assert torch.equal(embedding.embed(ids, weight, scale, out_dtype=o), want)


def test_lookup_of_views(hip_device):
    """Ids of any strides, a matrix with a row stride and an odd start."""
    gen = torch.Generator(hip_device).manual_seed(1)
    store = torch.randn(200 * 77 + 3, device=hip_device, generator=gen).to(BF16)
    weight = store[3:].as_strided((200, 45), (77, 1))
    ids = torch.randint(0, 200, (6, 10), device=hip_device, generator=gen).t()[1:, ::2]
    out = embedding.embed(ids, weight)
    assert out.shape == (9, 3, 45) and out.dtype == BF16 and torch.equal(out, weight[ids])
    assert embedding.embed(torch.tensor(5, device=hip_device), weight).shape == (45,)
    assert embedding.embed(ids[:0], weight).shape == (0, 3, 45)


@pytest.mark.parametrize("kind", ["random", "same", "few", "outside", "padded", "sorted"])
@pytest.mark.parametrize("n", [0, 1, 2, 31, 32, 33, 65, 4099, 8192, 8193, 20000])
def test_gradient_of_any_count(hip_device, kind, n):
    gen = torch.Generator(hip_device).manual_seed(n)
    vocab, dim = 1009, 40
    ids = make_ids(kind, n, vocab, gen, hip_device)
    dy = torch.randn(n, dim, device=hip_device, generator=gen).to(BF16)
    got = embedding.embedding_grad(ids, dy, vocab, scale=2.5)
    check_grad(got, ids, dy, 2.5)
    assert torch.equal(got, embedding.embedding_grad(ids, dy, vocab, scale=2.5))


@pytest.mark.parametrize("vocab", [1, 2, 255, 256, 49152, 65535, 65536, 70001])
@pytest.mark.parametrize("n", [100, 9000])
def test_gradient_of_any_vocabulary(hip_device, vocab, n):
    gen = torch.Generator(hip_device).manual_seed(vocab + n)
    ids = make_ids("random", n, vocab, gen, hip_device, torch.int32)
    dy = torch.randn(n, 24, device=hip_device, generator=gen)
    check_grad(embedding.embedding_grad(ids, dy, vocab, dtype=BF16), ids, dy, 1.0)


@pytest.mark.parametrize("dim", [1, 5, 8, 511, 512, 513, 649, 1280])
@pytest.mark.parametrize("g,w", [(BF16, FP32), (FP32, FP32), (BF16, BF16), (FP32, BF16)])
def test_gradient_of_any_width(hip_device, dim, g, w):
    gen = torch.Generator(hip_device).manual_seed(dim)
    ids = make_ids("few", 700, 300, gen, hip_device)
    ids[:300] = torch.randperm(300, device=hip_device, generator=gen)
    dy = torch.randn(700, dim, device=hip_device, generator=gen).to(g)
    check_grad(embedding.embedding_grad(ids, dy, 300, scale=0.5, dtype=w), ids, dy, 0.5)


@pytest.mark.parametrize("w", [FP32, BF16])
@pytest.mark.parametrize("n", [50, 10000])
def test_gradient_added_to_another(hip_device, w, n):
    """The rows of the batch's tokens grow, the others keep their bits; a buffer
    with a row stride keeps what lies between its rows."""
    gen = torch.Generator(hip_device).manual_seed(n)
    store = torch.randn(400, 50, device=hip_device, generator=gen).to(w)
    before, out = store.clone(), store[:, 2:45]
    ids = make_ids("few", n, 400, gen, hip_device)
    ids[0], ids[1] = 399, -100
    dy = torch.randn(n, 43, device=hip_device, generator=gen)
    version = out._version
    assert embedding.embedding_grad(ids, dy, 400, out=out, accumulate=True) is out and out._version > version
    check_grad(out, ids, dy, 1.0, old=before[:, 2:45])
    assert torch.equal(store[:, :2], before[:, :2]) and torch.equal(store[:, 45:], before[:, 45:])
    embedding.embedding_grad(ids, dy, 400, out=out)
    check_grad(out, ids, dy, 1.0)
    assert torch.equal(store[:, :2], before[:, :2]) and torch.equal(store[:, 45:], before[:, 45:])


def test_gradient_of_unaligned_memory(hip_device):
    gen = torch.Generator(hip_device).manual_seed(2)
    ids = make_ids("random", 333, 90, gen, hip_device)
    dy = torch.randn(333 * 31 + 1, device=hip_device, generator=gen).to(BF16)[1:].view(333, 31)
    out = torch.full((90 * 31 + 2,), 7.0, device=hip_device, dtype=BF16)
    embedding.embedding_grad(ids, dy, 90, out=out[1:-1].view(90, 31))
    check_grad(out[1:-1].view(90, 31), ids, dy, 1.0)
    assert out[0] == 7 and out[-1] == 7


def test_padding_row_takes_no_gradient(hip_device):
    gen = torch.Generator(hip_device).manual_seed(3)
    ids = make_ids("few", 100, 10, gen, hip_device)
    dy = torch.randn(100, 16, device=hip_device, generator=gen)
    for padding in (2, -8):
        check_grad(embedding.embedding_grad(ids, dy, 10, padding_idx=padding), ids, dy, 1.0, skip=2)


def test_module_matches_torch_module(hip_device):
    """Forward, gradient and a recorded backward's gradient against nn.Embedding."""
    torch.manual_seed(0)
    mine = embedding.Embedding(60, 24, padding_idx=5, device=hip_device)
    ref = torch.nn.Embedding(60, 24, padding_idx=5, device=hip_device)
    ref.load_state_dict(mine.state_dict())
    ids = torch.randint(0, 60, (4, 33), device=hip_device)
    ids[0, :3] = 5
    v = torch.randn(4, 33, 24, device=hip_device)
    assert torch.equal(mine(ids), ref(ids))
    seconds = []
    for m in (mine, ref):
        y = (m(ids) * v).sin()
        (g,) = torch.autograd.grad(y.sum(), m.weight, create_graph=True)
        (gg,) = torch.autograd.grad(g.square().sum(), m.weight)
        seconds.append((g.detach(), gg))
    # sums of at most 132 terms of magnitude up to |v| in both, in another order
    for a, b in zip(*seconds):
        assert (a - b).abs().max() <= 264 * 2.0 ** -24 * 8 * b.abs().max()
    assert not seconds[0][0][5].any()


def test_scaled_half_output_and_broadcast_gradient(hip_device):
    m = embedding.Embedding(50, 16, scale=4.0, out_dtype=BF16, device=hip_device)
    ids = torch.randint(0, 50, (7, 5), device=hip_device)
    y = m(ids)
    assert y.dtype == BF16 and torch.equal(y, (m.weight[ids] * 4).to(BF16))
    y.sum().backward()          # one gradient value expanded over all
    want = torch.bincount(ids.reshape(-1), minlength=50).float()[:, None] * 4
    assert torch.equal(m.weight.grad, want.expand(50, 16))
    with torch.no_grad():
        assert not m(ids).requires_grad


def test_tied_head_and_embedding_share_the_gradient(hip_device):
    """LMHead on an Embedding: the matrix's gradient is the sum of both uses,
    and equals the head's with the embedding's added to it in place."""
    torch.manual_seed(1)
    emb = embedding.Embedding(256, 128, out_dtype=BF16, device=hip_device)
    head = lm_head.LMHead(lm_head.HeadConfig(d_model=128, vocab=256), emb)
    ids = torch.randint(0, 256, (2, 60), device=hip_device)
    targets = torch.randint(0, 256, (2, 60), device=hip_device)
    hidden = emb(ids)
    head(hidden, targets).backward()
    both = emb.weight.grad.clone()
    emb.weight.grad = None
    free = hidden.detach().requires_grad_(True)
    head(free, targets).backward()
    embedding.embedding_grad(ids, free.grad, 256, out=emb.weight.grad, accumulate=True)
    # the two orders of one addition differ by a rounding
    assert (both - emb.weight.grad).abs().max() <= 2 * 2.0 ** -24 * both.abs().max()


def test_captured_and_replayed(hip_device):
    """Forward and gradient in a graph, replayed on new inputs between eager
    work, each replay equal to the eager call."""
    gen = torch.Generator(hip_device).manual_seed(4)
    for n in (100, 9000):
        weight = torch.randn(3000, 136, device=hip_device, generator=gen)
        ids = make_ids("random", n, 3000, gen, hip_device)
        dy = torch.randn(n, 136, device=hip_device, generator=gen).to(BF16)
        side = torch.cuda.Stream(hip_device)
        with torch.cuda.stream(side):
            embedding.embed(ids, weight), embedding.embedding_grad(ids, dy, 3000)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, grad = embedding.embed(ids, weight, out_dtype=BF16), embedding.embedding_grad(ids, dy, 3000)
        for k in range(4):
            ids.copy_(make_ids(("padded", "same", "few", "random")[k], n, 3000, gen, hip_device))
            dy.normal_(generator=gen)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, embedding.embed(ids, weight, out_dtype=BF16))
            assert torch.equal(grad, embedding.embedding_grad(ids, dy, 3000))


def test_two_streams_at_once(hip_device):
    """Two gradients in flight have workspaces of their own."""
    gen = torch.Generator(hip_device).manual_seed(5)
    sets = [(make_ids("random", 20000, 5000, gen, hip_device), torch.randn(20000, 64, device=hip_device, generator=gen))
            for _ in range(2)]
    want = [embedding.embedding_grad(i, d, 5000) for i, d in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(hip_device) for _ in sets]
    got = []
    for s, (i, d) in zip(streams, sets):
        with torch.cuda.stream(s):
            got.append([embedding.embedding_grad(i, d, 5000) for _ in range(4)])
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, t) for t in g)


def test_refusals(hip_device):
    ids = torch.zeros(4, dtype=torch.int64, device=hip_device)
    w = torch.zeros(10, 8, device=hip_device)
    dy = torch.zeros(4, 8, device=hip_device)
    for bad, error in [
        (lambda: embedding.embed(ids.float(), w), TypeError), (lambda: embedding.embed(ids.cpu(), w), ValueError),
        (lambda: embedding.embed(ids, w.cpu()), ValueError), (lambda: embedding.embed(ids, w.half()), TypeError),
        (lambda: embedding.embed(ids, w[0]), ValueError), (lambda: embedding.embed(ids, w.t()), ValueError),
        (lambda: embedding.embed(ids, w[:1].expand(10, 8)), ValueError),
        (lambda: embedding.embed(ids, w, out_dtype=torch.float16), TypeError),
        (lambda: embedding.embed(ids, w, padding_idx=10), ValueError),
        (lambda: embedding.embedding_grad(ids, dy[:3], 10), ValueError),
        (lambda: embedding.embedding_grad(ids, dy.double(), 10), TypeError),
        (lambda: embedding.embedding_grad(ids, dy, 0), ValueError),
        (lambda: embedding.embedding_grad(ids, dy, 10, accumulate=True), ValueError),
        (lambda: embedding.embedding_grad(ids, dy, 10, out=w.t()), ValueError),
        (lambda: embedding.embedding_grad(ids, dy, 11, out=w), ValueError),
        (lambda: embedding.embedding_grad(ids, dy, 10, out=w.clone().requires_grad_(True)), ValueError),
    ]:
        with pytest.raises(error):
            bad()


def test_sizes_past_the_librarys(hip_device):
    """Refused before anything is allocated."""
    ids, dy = torch.zeros(4, dtype=torch.int64, device=hip_device), torch.zeros(4, 1, device=hip_device)
    wide = torch.zeros(1, device=hip_device, dtype=BF16).expand((1 << 32) + 10, 1)
    for bad in (lambda: embedding.embedding_grad(ids, dy, (1 << 32) + 10), lambda: embedding.embed(ids, wide)):
        with pytest.raises(ValueError, match="rows are taken"):
            bad()


def test_gradient_into_its_inputs_memory_is_refused(hip_device):
    """Clearing or writing the matrix would change what the sums still read; other
    columns of the same rows are memory of their own."""
    gen = torch.Generator(hip_device).manual_seed(12)
    store = torch.randn(300, 96, device=hip_device, generator=gen)
    ids = make_ids("random", 300, 200, gen, hip_device)
    before = store.clone()
    for accumulate in (False, True):
        for out, dy in ((store[:200, :40], store[:, :40]), (store[:200, :40], store[:, 39:79]),
                        (store[100:, :40], store.view(-1)[:12000].view(300, 40)), (store[:200, :40], store[7, :40].expand(300, 40))):
            with pytest.raises(ValueError, match="share memory"):
                embedding.embedding_grad(ids, dy, 200, out=out, accumulate=accumulate)
        inside = store.view(torch.int64)[:200, 0]
        with pytest.raises(ValueError, match="share memory"):
            embedding.embedding_grad(inside, store[:200, 40:80], 200, out=store[:200, :40], accumulate=accumulate)
    assert torch.equal(store, before)
    store.view(torch.int64)[:, 47] = ids
    embedding.embedding_grad(store.view(torch.int64)[:, 47], store[:, 40:80], 200, out=store[:200, :40])
    check_grad(store[:200, :40], ids, before[:, 40:80], 1.0)
    assert torch.equal(store[:, 40:94], before[:, 40:94]) and torch.equal(store[200:, :94], before[200:, :94])


# The sort takes several workgroups from 16,385 tokens on, units of 32 tokens there and of 48 from
# 32,769 on, and passes' counts in global memory from 524,289 on (65 tiles of 8192).
@pytest.mark.parametrize("kind", ["random", "same", "few", "outside", "padded", "sorted"])
@pytest.mark.parametrize("n", [16384, 16385, 32768, 32769, 50021])
def test_gradient_where_the_sort_changes(hip_device, kind, n):
    gen = torch.Generator(hip_device).manual_seed(n)
    ids = make_ids(kind, n, 1009, gen, hip_device)
    dy = torch.randn(n, 40, device=hip_device, generator=gen).to(BF16)
    got = embedding.embedding_grad(ids, dy, 1009, scale=2.5)
    check_grad(got, ids, dy, 2.5)
    assert torch.equal(got, embedding.embedding_grad(ids, dy, 1009, scale=2.5))


@pytest.mark.parametrize("vocab", [1, 2, 255, 256, 49152, 65535, 65536, 70001])
@pytest.mark.parametrize("n", [20000, 40000])
def test_gradient_of_any_vocabulary_by_several_workgroups(hip_device, vocab, n):
    """One, two and three passes of the sort over several tiles."""
    gen = torch.Generator(hip_device).manual_seed(vocab + n)
    ids = make_ids("random", n, vocab, gen, hip_device, torch.int32)
    dy = torch.randn(n, 24, device=hip_device, generator=gen)
    check_grad(embedding.embedding_grad(ids, dy, vocab, dtype=BF16), ids, dy, 1.0)


@pytest.mark.parametrize("w", [FP32, BF16])
@pytest.mark.parametrize("vocab,kind", [(200, "random"), (400, "few"), (70001, "random"), (70001, "same")])
def test_gradient_added_by_several_workgroups(hip_device, w, vocab, kind):
    """Added to a buffer with a row stride, and written over it, its rows cleared
    piece by piece beside the passes."""
    n = 20011
    gen = torch.Generator(hip_device).manual_seed(vocab)
    store = torch.randn(vocab, 50, device=hip_device, generator=gen).to(w)
    before, out = store.clone(), store[:, 2:45]
    ids = make_ids(kind, n, vocab, gen, hip_device)
    ids[0], ids[1], ids[n - 1] = vocab - 1, -100, vocab
    dy = torch.randn(n, 43, device=hip_device, generator=gen)
    embedding.embedding_grad(ids, dy, vocab, out=out, accumulate=True)
    check_grad(out, ids, dy, 1.0, old=before[:, 2:45])
    assert torch.equal(store[:, :2], before[:, :2]) and torch.equal(store[:, 45:], before[:, 45:])
    embedding.embedding_grad(ids, dy, vocab, out=out)
    check_grad(out, ids, dy, 1.0)
    assert torch.equal(store[:, :2], before[:, :2]) and torch.equal(store[:, 45:], before[:, 45:])


@pytest.mark.parametrize("vocab", [200, 3000, 70001])
def test_several_workgroups_captured_and_replayed(hip_device, vocab):
    gen = torch.Generator(hip_device).manual_seed(vocab)
    n = 20000
    ids = make_ids("random", n, vocab, gen, hip_device)
    dy = torch.randn(n, 24, device=hip_device, generator=gen)
    kept = torch.randn(vocab, 24, device=hip_device, generator=gen)
    old = kept.clone()
    side = torch.cuda.Stream(hip_device)
    with torch.cuda.stream(side):
        embedding.embedding_grad(ids, dy, vocab)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad = embedding.embedding_grad(ids, dy, vocab)
        embedding.embedding_grad(ids, dy, vocab, out=kept, accumulate=True)
    for kind in ("padded", "same", "few", "random"):
        ids.copy_(make_ids(kind, n, vocab, gen, hip_device))
        dy.normal_(generator=gen)
        kept.copy_(old)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, embedding.embedding_grad(ids, dy, vocab))
        assert torch.equal(kept, embedding.embedding_grad(ids, dy, vocab, out=old.clone(), accumulate=True))


@pytest.mark.parametrize("vocab", [200, 1009, 70001])
@pytest.mark.parametrize("kind", ["random", "few", "padded"])
def test_gradient_of_more_tiles_than_counts_in_lds(hip_device, vocab, kind):
    """Runs of a frequent id over thousands of units; the passes count the next
    one's digits in global memory."""
    n = 530_003
    gen = torch.Generator(hip_device).manual_seed(vocab)
    ids = make_ids(kind, n, vocab, gen, hip_device)
    dy = torch.randn(n, 8, device=hip_device, generator=gen)
    got = embedding.embedding_grad(ids, dy, vocab)
    check_grad(got, ids, dy, 1.0)
    assert torch.equal(got, embedding.embedding_grad(ids, dy, vocab))


@pytest.mark.parametrize("w", [FP32, BF16])
def test_rows_past_32_bit_offsets(hip_device, w):
    """A matrix, and a batch, of more than 2^31 values: lookup and gradient at both ends."""
    vocab, dim, n = 2_200_003, 1000, 3000
    gen = torch.Generator(hip_device).manual_seed(6)
    weight = torch.empty(vocab, dim, device=hip_device, dtype=w).normal_(generator=gen)
    ids = torch.cat([torch.randint(0, 100, (n // 2,), generator=gen, device=hip_device),
                     torch.randint(vocab - 1000, vocab, (n - n // 2,), generator=gen, device=hip_device)])
    assert torch.equal(embedding.embed(ids, weight), weight[ids])
    dy = torch.randn(n, dim, device=hip_device, generator=gen)
    grad = embedding.embedding_grad(ids, dy, vocab, out=weight)
    low, high = grad[:100].clone(), grad[vocab - 1000:].clone()
    assert not grad[100:vocab - 1000].any()
    outside = torch.where(ids < 100, ids, -1)
    check_grad(low, outside, dy, 1.0)
    check_grad(high, torch.where(ids >= 100, ids - (vocab - 1000), -1), dy, 1.0)
    del weight, grad
    small = torch.randn(50, dim, device=hip_device, generator=gen).to(w)
    many = torch.randint(0, 50, (vocab,), generator=gen, device=hip_device)
    y = embedding.embed(many, small, out_dtype=BF16)
    for part in (slice(0, 1000), slice(vocab - 1000, vocab)):
        assert torch.equal(y[part], small[many[part]].to(BF16))
    # the sums read rows past 2^31 values: a token counts where its id is in range
    many[1000:vocab - 1000] = -1
    got = embedding.embedding_grad(many, y, 50)
    check_grad(got, torch.cat([many[:1000], many[vocab - 1000:]]), torch.cat([y[:1000], y[vocab - 1000:]]), 1.0)
    del y
    torch.cuda.empty_cache()


def test_gradient_of_the_most_tokens(hip_device):
    """2^26 tokens, the most that are taken, a quarter of them the same one, against
    64-bit sums on the host."""
    n, vocab = 1 << 26, 70001
    gen = torch.Generator(hip_device).manual_seed(7)
    ids = (torch.rand(n, device=hip_device, generator=gen) ** 8 * vocab).int().clamp(max=vocab - 1)
    dy = torch.randn(n, 1, device=hip_device, generator=gen)
    got = embedding.embedding_grad(ids, dy, vocab)[:, 0].cpu().numpy()
    index, terms = ids.cpu().numpy(), dy[:, 0].double().cpu().numpy()
    want, size = np.bincount(index, terms, vocab), np.bincount(index, np.abs(terms), vocab)
    count = np.bincount(index, minlength=vocab)
    assert (np.abs(got - want) <= (count + 3) * 2.0 ** -24 * 1.01 * size).all()
    more = torch.zeros(n + 1, dtype=torch.int32, device=hip_device)
    with pytest.raises(_lib.AttnError):
        embedding.embedding_grad(more, dy[:1].expand(n + 1, 1), vocab)
    del ids, dy, more
    torch.cuda.empty_cache()
