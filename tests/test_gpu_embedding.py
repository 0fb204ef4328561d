"""embedding_lookup and its gradient (dg_embedding_lookup, dg_embedding_grad) against the formulas in 64 bits.

    Y[i] = s E[t_i]     dE[v] = s sum over i with t_i = v of G[i]

Tolerances, from the arithmetic (u = 2^-24, half a step of fp32; h = half a step of the table's type):
  Y   the scale rounds to fp32 once (u), the product once (u), the result once (h): |Y| (h + 2 u), and half of the smallest
      subnormal where fp16 results underflow
  dE  k - 1 additions of k fp32 numbers in any order: at most (k - 1) u sum|G| (to first order; 1 % covers the rest), the
      scale and its product 2 u more, the result h: 1.01 (k + 2) u |s| sum|G| + h |dE|"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = {torch.float16: 2.0 ** -25, torch.float32: 0.0, torch.bfloat16: 0.0}


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _case(dev, v, d, n, dtype, index, seed=0, hot=None):
    g = torch.Generator().manual_seed(seed)
    table = torch.randn((v, d), generator=g).to(dtype).to(dev)
    tokens = torch.randint(0, v, (n,), generator=g)
    if hot is not None and n:
        tokens[torch.rand(n, generator=g) < hot] = v // 2
    grad = torch.randn((n, d), generator=g).to(dtype).to(dev)
    return table, tokens.to(index).to(dev), grad


def _check_lookup(out, table, tokens, scale):
    want = table.double()[tokens.long()] * scale
    tol = want.abs() * (_half(table.dtype) + 2 * U) + TINY[table.dtype]
    assert out.dtype == table.dtype and out.shape == want.shape
    assert bool(((out.double() - want).abs() <= tol).all())


def _check_grad(got, grad, tokens, scale, v, padding=None):
    t = tokens.reshape(-1).long().cpu()
    g = grad.reshape(t.numel(), grad.shape[-1]).double().cpu()
    d = g.shape[1]
    keep = (t >= 0) & (t < v)
    if padding is not None:
        keep &= t != padding
    t, g = t[keep], g[keep]
    want = torch.zeros((v, d), dtype=torch.float64).index_add_(0, t, g) * scale
    size = torch.zeros((v, d), dtype=torch.float64).index_add_(0, t, g.abs()) * abs(scale)
    k = torch.bincount(t, minlength=v).double()[:, None]
    tol = 1.01 * (k + 2) * U * size + _half(grad.dtype) * want.abs() + TINY[grad.dtype]
    got = got.double().cpu()
    assert got.shape == want.shape
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() - tol).max())


SIZES = [  # rows, width, tokens, share of one hot token
    (1, 1, 1, None), (3, 5, 0, None), (1, 64, 1000, None), (7, 1, 100, None), (64, 64, 1, None), (300, 64, 257, None),
    (1000, 100, 4097, 0.5), (50, 1023, 1000, None), (500, 4100, 300, None), (2, 8, 20000, None), (131072, 16, 5000, 0.3),
    (40000, 33, 20001, 0.9), (1000, 2048, 3000, 0.2), (65537, 7, 70000, 0.05), (255, 129, 16384, None), (33, 9000, 65, None),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("v,d,n,hot", SIZES)
def test_lookup_and_gradient(hip_device, v, d, n, hot, dtype):
    from dogs_amd.embedding import embedding_lookup
    index = torch.int64 if (v + n) % 2 else torch.int32
    table, tokens, grad = _case(hip_device, v, d, n, dtype, index, seed=v + d + n, hot=hot)
    scale = math.sqrt(d)
    table.requires_grad_(True)
    out = embedding_lookup(table, tokens, scale=scale)
    _check_lookup(out.detach(), table.detach(), tokens, scale)
    out.backward(grad)
    assert table.grad.dtype == dtype and table.grad.is_contiguous()
    _check_grad(table.grad, grad, tokens, scale, v)
    first = table.grad
    table.grad = None
    embedding_lookup(table, tokens, scale=scale).backward(grad)
    assert torch.equal(first, table.grad)      # the same bits each time
    with torch.no_grad():
        assert torch.equal(embedding_lookup(table, tokens, scale=scale), out)


def test_every_length_around_the_variants(hip_device):
    """Row counts, widths and lengths on either side of what chooses a variant; one token alone, and all alike."""
    from dogs_amd.embedding import embedding_lookup
    for n in (1, 2, 63, 64, 65, 255, 256, 257, 1023, 1024, 1025, 2047, 2048, 2049, 4095, 4096, 4097, 8191, 8192, 8193, 16385, 32769):
        for v, d in ((n % 7 + 1, 24), (2000, 10)):
            for hot in (None, 1.1):
                table, tokens, grad = _case(hip_device, v, d, n, torch.float32, torch.int64, seed=n, hot=hot)
                table.requires_grad_(True)
                out = embedding_lookup(table, tokens, scale=0.5)
                out.backward(grad)
                _check_lookup(out.detach(), table.detach(), tokens, 0.5)
                _check_grad(table.grad, grad, tokens, 0.5, v)


@pytest.mark.parametrize("v,d,n,hot", [
    (1, 600, 3000, None), (2, 300, 8000, None), (3, 517, 7000, 0.5), (1, 2, 8192, None),      # few rows with long lists
    (1, 3, 20000, None), (5_000_000, 2, 9000, 0.2), (2 ** 22, 3, 9000, None), (2 ** 22 - 1, 3, 9000, None),    # 1, 2, 3 sort passes
    (1000, 3, 2 ** 18, 0.3), (1000, 3, 2 ** 18 + 1, 0.3), (3_000_000, 5, 300_000, 0.5), (3, 1, 600_000, None)])
def test_long_lists(hip_device, v, d, n, hot):
    """Lists on either side of what the wide-digit sort takes, tables of many rows, one row that all tokens share."""
    from dogs_amd.embedding import embedding_lookup
    table, tokens, grad = _case(hip_device, v, d, n, torch.bfloat16, torch.int64, seed=v % 97 + n, hot=hot)
    table.requires_grad_(True)
    out = embedding_lookup(table, tokens, scale=0.75, padding_idx=0 if v > 1 else None)
    _check_lookup(out.detach(), table.detach(), tokens, 0.75)
    out.backward(grad)
    _check_grad(table.grad, grad, tokens, 0.75, v, 0 if v > 1 else None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("v,d,n,hot", [
    (2, 300, 8000, None), (2 ** 22, 3, 9000, 0.2), (1000, 3, 2 ** 18, 0.3), (700, 37, 2 ** 18 + 1, 0.3), (200_000, 65, 300_000, None)])
def test_long_lists_of_other_types(hip_device, v, d, n, hot, dtype):
    from dogs_amd.embedding import embedding_lookup
    table, tokens, grad = _case(hip_device, v, d, n, dtype, torch.int32, seed=v % 89 + n, hot=hot)
    table.requires_grad_(True)
    out = embedding_lookup(table, tokens, scale=0.25, padding_idx=1)
    _check_lookup(out.detach(), table.detach(), tokens, 0.25)
    out.backward(grad)
    _check_grad(table.grad, grad, tokens, 0.25, v, 1)


def test_long_list_in_a_graph(hip_device):
    """The sort of more than 2^18 tokens, captured: several replays with other tokens and eager work between them."""
    from dogs_amd.embedding import embedding_lookup
    v, n = 3000, 2 ** 18 + 77
    table, tokens, grad = _case(hip_device, v, 9, n, torch.float32, torch.int64, seed=12)
    table.requires_grad_(True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dt, = torch.autograd.grad(embedding_lookup(table, tokens), table, grad)
    for k in range(3):
        g = torch.Generator().manual_seed(60 + k)
        tokens.copy_(torch.randint(0, v >> k, (n,), generator=g))
        grad.copy_(torch.randn((n, 9), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = dt.clone()
        _check_grad(got, grad, tokens, 1.0, v)
        eager, = torch.autograd.grad(embedding_lookup(table, tokens), table, grad)
        assert torch.equal(got, eager)


@pytest.mark.parametrize("n", [9, 700, 30000])
@pytest.mark.parametrize("padding", [0, 17, -1])
def test_padding_row_gets_no_gradient(hip_device, padding, n):
    from dogs_amd.embedding import embedding_lookup
    v = 18 + n % 3
    table, tokens, grad = _case(hip_device, v, 40, n, torch.float32, torch.int64, seed=n)
    tokens[::2] = padding % v
    table.requires_grad_(True)
    out = embedding_lookup(table, tokens, padding_idx=padding)
    _check_lookup(out.detach(), table.detach(), tokens, 1.0)   # the padding row is read like any other
    out.backward(grad)
    _check_grad(table.grad, grad, tokens, 1.0, v, padding % v)
    assert not table.grad[padding % v].any()


@pytest.mark.parametrize("n", [12, 5000])
def test_tokens_out_of_range(hip_device, n):
    """On the device: a NaN row, and nothing added.  On the host: an IndexError."""
    from dogs_amd.embedding import embedding_lookup
    v, d = 37, 20
    table, tokens, grad = _case(hip_device, v, d, n, torch.float32, torch.int64, seed=1)
    bad = [-1, v, 2 ** 40, -2 ** 63, 2 ** 32 + 3, 2 ** 31]
    tokens[:6] = torch.tensor(bad, device=hip_device)
    table.requires_grad_(True)
    out = embedding_lookup(table, tokens)
    assert bool(out[:6].isnan().all())
    _check_lookup(out[6:].detach(), table.detach(), tokens[6:], 1.0)
    out.backward(grad)
    _check_grad(table.grad, grad, tokens, 1.0, v)
    for t in ([0, -1], [v]):
        with pytest.raises(IndexError):
            embedding_lookup(table, torch.tensor(t))
    host = torch.tensor([3, v - 1, 0], dtype=torch.int32)
    _check_lookup(embedding_lookup(table, host).detach(), table.detach(), host.to(hip_device), 1.0)


def test_infinities_and_nan_stay_in_their_rows(hip_device):
    from dogs_amd.embedding import embedding_lookup
    for n in (40, 9000):
        table, tokens, grad = _case(hip_device, 30, 16, n, torch.float32, torch.int64, seed=2)
        table[4], table[5] = math.inf, math.nan
        grad[0, 0], grad[1, 1] = math.inf, math.nan
        table.requires_grad_(True)
        out = embedding_lookup(table, tokens, scale=2.0)
        want = table.detach()[tokens] * 2.0
        assert torch.equal(out.detach().nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0))
        out.backward(grad)
        want = torch.zeros((30, 16), dtype=torch.float64).index_add_(0, tokens.cpu(), grad.double().cpu())
        assert torch.equal(table.grad.cpu().isfinite(), want.isfinite())
        assert torch.equal(table.grad.cpu().isnan(), want.isnan())


def test_strides(hip_device):
    """Tables that are slices, transposed or broadcast; tokens and gradients that are not contiguous."""
    from dogs_amd.embedding import embedding_lookup
    g = torch.Generator().manual_seed(3)
    base = torch.randn((60, 90), generator=g).to(torch.bfloat16).to(hip_device)
    tokens = torch.randint(0, 25, (40, 6), generator=g).to(hip_device)
    for table in (base[3:33, 1:72], base.t()[5:40, 3:44], base[:30, ::3], base[:1, :33].expand(28, 33), base[1::2, :65]):
        out = embedding_lookup(table, tokens.t(), scale=1.5)
        assert out.shape == (6, 40, table.shape[1])
        _check_lookup(out, table, tokens.t(), 1.5)
    leaf = base[:30, :41].float().clone().requires_grad_(True)
    out = embedding_lookup(leaf.t().contiguous().t(), tokens[:, ::2], scale=1.5)
    wide = torch.randn((40, 41, 3), generator=g).to(hip_device).transpose(1, 2)
    out.backward(wide)
    _check_grad(leaf.grad, wide.reshape(-1, 41), tokens[:, ::2], 1.5, 30)
    leaf.grad = None
    embedding_lookup(leaf, tokens).sum().backward()        # a gradient of stride 0
    _check_grad(leaf.grad, torch.ones((240, 41)), tokens, 1.0, 30)
    slim = base[:30].float().clone().requires_grad_(True)   # a leaf seen through a view
    embedding_lookup(slim[:, 7:48], tokens[0]).sum().backward()
    want = torch.zeros((30, 90))
    want[:, 7:48] = torch.bincount(tokens[0].cpu(), minlength=30)[:, None].float()
    assert torch.equal(slim.grad.cpu(), want)


def test_negated_views(hip_device):
    """Views whose memory holds the other sign (a conjugate's imaginary part): as a table, contiguous or strided, one that
    learns, and as the result's gradient."""
    from dogs_amd.embedding import embedding_lookup
    g = torch.Generator().manual_seed(8)
    tokens = torch.tensor([1, 1, 5], device=hip_device)
    z = torch.complex(torch.randn((6, 8), generator=g), torch.randn((6, 8), generator=g)).to(hip_device)
    for view, want in ((z.conj().imag, -z.imag), (torch._neg_view(z.real.contiguous()), -z.real)):
        assert view.is_neg()
        assert torch.equal(embedding_lookup(view, tokens), want[tokens])
        leaf = view.detach().requires_grad_(True)
        out = embedding_lookup(leaf, tokens)
        assert torch.equal(out, want[tokens])
        out[0].sum().backward()
        assert torch.equal(leaf.grad[:, 0].cpu(), torch.tensor([0.0, 1.0, 0.0, 0.0, 0.0, 0.0]))
    table = torch.randn((6, 8), generator=g).to(hip_device).requires_grad_(True)
    out = embedding_lookup(table, tokens)
    up = torch.randn((3, 8), generator=g).to(hip_device)
    a, = torch.autograd.grad(out, table, torch._neg_view(up), retain_graph=True)
    b, = torch.autograd.grad(out, table, -up)
    assert torch.equal(a, b)


def test_gradient_against_differences(hip_device):
    """The lookup is linear: on small whole numbers and a power of two as scale every product and sum here is exact, so a
    difference of the loss equals the gradient's product with the step to the last bit."""
    from dogs_amd.embedding import embedding_lookup
    g = torch.Generator().manual_seed(4)
    for n in (50, 3000):
        table = torch.randint(-8, 9, (20, 12), generator=g).float().to(hip_device).requires_grad_(True)
        step = torch.randint(-4, 5, (20, 12), generator=g).float().to(hip_device)
        tokens = torch.randint(0, 20, (n,), generator=g).to(hip_device)
        w = torch.randint(-3, 4, (n, 12), generator=g).float().to(hip_device)
        (embedding_lookup(table, tokens, scale=0.25) * w).sum().backward()

        def loss(e):
            return (embedding_lookup(e.detach(), tokens, scale=0.25).double() * w.double()).sum()
        assert float(loss(table + step) - loss(table)) == float((table.grad.double() * step.double()).sum())


def test_past_32_bit_offsets(hip_device):
    """Tables, results and gradients of more than 2^32 elements."""
    from dogs_amd.embedding import embedding_lookup
    v, d = 70001, 65536
    table = torch.empty((v, d), dtype=torch.bfloat16, device=hip_device)
    rows = [0, 1, 65536, 65537, 69999, 70000]
    for k, r in enumerate(rows):
        table[r] = float(k + 1)
    tokens = torch.tensor(rows * 11700, device=hip_device)                # 70200 rows of result
    out = embedding_lookup(table, tokens, scale=2.0)
    got = out[:, ::9999].float().cpu()
    assert torch.equal(got, (torch.arange(6) + 1).float().mul(2).repeat(11700)[:, None].expand_as(got))
    assert bool((out[-6:].float().amax(1) == out[-6:].float().amin(1)).all())
    table.requires_grad_(True)
    grad = out.fill_(1.0)
    again = embedding_lookup(table, tokens)
    again.backward(grad)
    total = table.grad[:, ::8191].float().cpu()
    want = torch.zeros_like(total)
    want[rows] = torch.tensor(11700.0).to(torch.bfloat16).float()
    assert torch.equal(total, want)
    assert bool((table.grad[rows].float() == want[0, 0]).all())


def test_side_stream_and_graph(hip_device):
    from dogs_amd.embedding import embedding_lookup
    side = torch.cuda.Stream()
    for n in (200, 9000):
        table, tokens, grad = _case(hip_device, 500, 48, n, torch.float32, torch.int64, seed=5)
        table.requires_grad_(True)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            out = embedding_lookup(table, tokens)
            dt, = torch.autograd.grad(out, table, grad)
        side.synchronize()
        _check_lookup(out.detach(), table.detach(), tokens, 1.0)
        _check_grad(dt, grad, tokens, 1.0, 500)
        del out, dt
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = embedding_lookup(table, tokens)
            z, = torch.autograd.grad(y, table, grad)
        y, z = y.detach(), z.detach()
        for k in range(4):
            g = torch.Generator().manual_seed(50 + k)
            with torch.no_grad():
                tokens.copy_(torch.randint(0, 500, (n,), generator=g))
                table.copy_(torch.randn((500, 48), generator=g))
                grad.copy_(torch.randn((n, 48), generator=g))
            graph.replay()
            with torch.no_grad():
                eager = embedding_lookup(table, tokens)
            assert torch.equal(y, eager)
            torch.cuda.synchronize()
            _check_grad(z, grad, tokens, 1.0, 500)


def test_second_derivative_is_refused(hip_device):
    from dogs_amd.embedding import embedding_lookup
    table = torch.randn((5, 4), device=hip_device, requires_grad=True)
    w = torch.ones((3, 4), device=hip_device, requires_grad=True)
    out = embedding_lookup(table, torch.tensor([0, 1, 1], device=hip_device))
    dt, = torch.autograd.grad((out * w).sum(), table, create_graph=True)
    with pytest.raises(RuntimeError):
        dt.sum().backward()


@pytest.mark.parametrize("learns", [False, True])
def test_forward_mode_is_refused(hip_device, learns):
    """A dual table, and a dual gradient of the result (forward over reverse): an error, not a derivative of zero."""
    import torch.autograd.forward_ad as fw

    from dogs_amd.embedding import embedding_lookup
    table = torch.randn((5, 4), device=hip_device, requires_grad=learns)
    tokens = torch.tensor([0, 3, 3], device=hip_device)
    with fw.dual_level():
        dual = fw.make_dual(table, torch.ones_like(table))
        with pytest.raises(RuntimeError, match="forward-mode"):
            embedding_lookup(dual, tokens)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            embedding_lookup(dual, tokens)
        out = embedding_lookup(table, tokens)      # what carries no tangent goes on
        assert torch.equal(out, table[tokens])
        if learns:
            g = torch.ones((3, 4), device=hip_device)
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, table, fw.make_dual(g, g))
            dt, = torch.autograd.grad(embedding_lookup(table, tokens), table, g)
            assert torch.equal(dt[:, 0].cpu(), torch.tensor([1.0, 0.0, 0.0, 2.0, 0.0]))


@pytest.mark.parametrize("learns", [False, True])
def test_tracing_is_refused(hip_device, learns):
    from dogs_amd.embedding import embedding_lookup
    table = torch.randn((5, 4), device=hip_device, requires_grad=learns)
    tokens = torch.tensor([0, 3, 3], device=hip_device)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda e: embedding_lookup(e, tokens), (table,))
    assert torch.equal(embedding_lookup(table, tokens), table[tokens])


def test_tokens_changed_before_the_backward_are_noticed(hip_device):
    from dogs_amd.embedding import embedding_lookup
    table = torch.randn((5, 4), device=hip_device, requires_grad=True)
    tokens = torch.tensor([0, 1, 1], device=hip_device)
    out = embedding_lookup(table, tokens)
    tokens.zero_()
    with pytest.raises(RuntimeError):
        out.sum().backward()


def test_refusals(hip_device):
    from dogs_amd.embedding import embedding_lookup
    table = torch.zeros((4, 4), device=hip_device)
    tok = torch.tensor([1], device=hip_device)
    for t, k in ((table.double(), tok), (table[0], tok), (table, tok.float()), (table, tok.bool()), (table.int(), tok)):
        with pytest.raises(RuntimeError):
            embedding_lookup(t, k)
    with pytest.raises(RuntimeError):
        embedding_lookup(table, tok, scale=torch.tensor(2.0, requires_grad=True))
    for p in (4, -5):
        with pytest.raises(IndexError):
            embedding_lookup(table, tok, padding_idx=p)


def test_empty(hip_device):
    from dogs_amd.embedding import embedding_lookup
    table = torch.randn((4, 6), device=hip_device, requires_grad=True)
    none = torch.empty((0, 3), dtype=torch.int64, device=hip_device)
    out = embedding_lookup(table, none)
    assert out.shape == (0, 3, 6)
    out.sum().backward()
    assert torch.equal(table.grad, torch.zeros_like(table))
    flat = torch.empty((4, 0), device=hip_device, requires_grad=True)
    out = embedding_lookup(flat, torch.tensor([1, 2], device=hip_device))
    assert out.shape == (2, 0)
    out.sum().backward()
    assert flat.grad.shape == (4, 0)
    bare = torch.empty((0, 6), device=hip_device, requires_grad=True)
    out = embedding_lookup(bare, none)
    out.sum().backward()
    assert bare.grad.shape == (0, 6)


@pytest.mark.parametrize("n", [2, 1025, 9000])
def test_table_without_columns(hip_device, n):
    from dogs_amd.embedding import embedding_lookup
    flat = torch.empty((4, 0), device=hip_device, requires_grad=True)
    out = embedding_lookup(flat, torch.zeros(n, dtype=torch.int64, device=hip_device))
    assert out.shape == (n, 0)
    out.sum().backward()
    assert flat.grad.shape == (4, 0)


def _network(dev, views):
    from dogs_amd.masks import AppearanceEmbedding
    torch.manual_seed(0)
    net = AppearanceEmbedding(views).to(dev)
    with torch.no_grad():
        net.appearance_embedding.normal_()
    return net


def test_appearance_batch_equals_the_single_views(hip_device):
    """AppearanceEmbedding over a batch: each mask has the bits of that view's own call; the table's gradient is the sum of
    the views' gradients, a view that is there twice adding both (three addends: two roundings)."""
    net = _network(hip_device, 9)
    g = torch.Generator().manual_seed(6)
    images = torch.rand((3, 3, 4, 5), generator=g).to(hip_device)
    index = torch.tensor([7, 2, 7], device=hip_device)
    w = torch.randn((3, 3, 100, 130), generator=g).to(hip_device)
    masks = net(images, index, (100, 130))
    (masks * w).sum().backward()
    got = net.appearance_embedding.grad.clone()
    parts = []
    for k in range(3):
        net.zero_grad()
        one = net(images[k], int(index[k]), (100, 130))
        assert torch.equal(one, masks[k])
        (one * w[k]).sum().backward()
        parts.append(net.appearance_embedding.grad.double().clone())
    want, size = sum(parts), sum(p.abs() for p in parts)
    # the code's gradient of one view is the same sum over its pixels, taken in another order: 20 addends
    assert bool(((got.double() - want).abs() <= 64 * U * size + 1e-6 * want.abs().max()).all())
    assert not got[[0, 1, 3, 4, 5, 6, 8]].any()
    assert torch.equal(net(images, index.cpu(), (100, 130)), masks)
    for bad in (3, [7, 2, 7], index[:2]):
        with pytest.raises(ValueError):
            net(images, bad, (100, 130))
    with pytest.raises(ValueError):
        net(images[:0], index[:0], (100, 130))


def test_batched_clipped_step(hip_device):
    """Batch lookup, network, backward, clipping and the step together, against the same step in plain torch."""
    from dogs_amd.gradclip import clip_grad_norm_
    net = _network(hip_device, 9)
    opt = torch.optim.SGD(net.parameters(), lr=0.1)
    g = torch.Generator().manual_seed(7)
    images = torch.rand((2, 3, 4, 5), generator=g).to(hip_device)
    index = torch.tensor([1, 8], device=hip_device)
    ((net(images, index, (64, 80)) - 1) ** 2).sum().backward()
    before = [p.detach().double() for p in net.parameters()]
    grads = [p.grad.double() for p in net.parameters()]
    n = math.sqrt(sum(float((x ** 2).sum()) for x in grads))
    limit = n / 3
    norm = clip_grad_norm_(net.parameters(), limit)
    assert abs(float(norm) - n) <= 2 * U * n
    opt.step()
    for p, b, x in zip(net.parameters(), before, grads):
        want = b - 0.1 * x * (limit / (n + 1e-6))
        # two roundings of the step's product, one more of the coefficient, one of the difference
        tol = 4 * U * (0.1 * x.abs() * (limit / n)) + 2 * U * want.abs() + 1e-30
        assert bool(((p.detach().double() - want).abs() <= tol).all())
