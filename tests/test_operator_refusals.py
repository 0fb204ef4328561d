"""What embedding_lookup, grad_norm, clip_grad_norm_ and the library's entries below them refuse, without a GPU: every call
here has to return an error before anything is launched."""
import ctypes as C
from array import array

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    import os

    from dogs_amd import _lib
    from dogs_amd import build as B
    if not os.path.exists(_lib.LIB_PATH):
        B.build()
    return _lib.load()


def test_host_tensors_are_refused():
    from dogs_amd.embedding import embedding_lookup
    from dogs_amd.gradclip import clip_grad_norm_, grad_norm
    with pytest.raises(RuntimeError):
        embedding_lookup(torch.zeros(4, 4), torch.tensor([1]))
    with pytest.raises(RuntimeError):
        grad_norm([torch.ones(3)])
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError):
        clip_grad_norm_([p], 1.0)


def test_embedding_entry_refusals(lib):
    def lookup(table=16, dtype=0, v=4, d=4, tokens=16, n=2, out=16):
        return lib.dg_embedding_lookup(table, dtype, v, d, d, 1, tokens, 1, n, 1.0, out, None)
    for kw in ({"dtype": 3}, {"dtype": -1}, {"v": 1 << 31}, {"n": 1 << 31}, {"d": 1 << 23}, {"table": None},
               {"tokens": None}, {"out": None}):
        assert lookup(**kw) != 0, kw
    assert lookup(n=0) == 0 and lookup(d=0) == 0

    def grad(g=16, dtype=0, v=4, d=4, tokens=16, n=2, out=16, scratch=256, nbytes=1 << 20):
        return lib.dg_embedding_grad(g, dtype, tokens, 1, n, v, d, 1.0, -1, out, scratch, nbytes, None)
    need = lib.dg_embedding_grad_scratch_bytes(4, 4, 20000, 0)
    assert need > 0
    for v in (1, 2, 1000, 1 << 20, (1 << 31) - 1):      # the Python side does not ask up to 1024 tokens
        for d in (1, 64, 4096, (1 << 23) - 1):
            for dtype in (0, 1, 2):
                assert lib.dg_embedding_grad_scratch_bytes(v, d, 1024, dtype) == 0
    for kw in ({"dtype": 3}, {"v": 1 << 31}, {"n": 1 << 31}, {"d": 1 << 23}, {"g": None}, {"tokens": None}, {"out": None},
               {"n": 20000, "scratch": None}, {"n": 20000, "nbytes": need - 1}):
        assert grad(**kw) != 0, kw
    assert grad(v=0) == 0 and grad(d=0) == 0
    assert lib.dg_embedding_grad_scratch_bytes(1 << 31, 4, 2, 0) == 0


def test_scratch_of_empty_and_refused_sizes(lib):
    """A table without rows or columns needs no scratch, however long the list (the row's bytes divide nothing), and sizes
    that the gradient refuses are not priced."""
    for n in (1, 1024, 1025, 8192, 8193, 9000, 300_000, (1 << 31) - 1):
        for dtype in (0, 1, 2):
            for v, d in ((4, 0), (0, 4), (0, 0), ((1 << 31) - 1, 0), (4, 1 << 23), (4, (1 << 32) - 1)):
                assert lib.dg_embedding_grad_scratch_bytes(v, d, n, dtype) == 0, (v, d, n, dtype)
    assert lib.dg_embedding_grad(16, 0, 16, 1, 9000, 4, 0, 1.0, -1, 16, None, 0, None) == 0


def test_gradient_entry_refusals(lib):
    def args(ptrs, sizes, types):
        keep = array("Q", ptrs), array("Q", sizes), array("B", types)
        return keep, (len(ptrs), *[k.buffer_info()[0] for k in keep])
    need = lib.dg_grad_norm_scratch_bytes(2)
    for ptrs, sizes, types, text in (
            ((4096, 4096), (10, 10), (0, 0), b"overlap"), ((4096, 4100), (10, 10), (0, 0), b"overlap"),
            ((8192, 4096), (1, 1025), (0, 0), b"overlap"), ((4096, 8192), (2049, 1), (2, 2), b"overlap"),
            ((4096, 8192), (1, 1), (0, 3), b"element type"), ((4096, 0), (1, 1), (0, 0), b"NULL"),
            ((4096, 8194), (1, 1), (0, 0), b"aligned"), ((4096, 8193), (1, 1), (0, 2), b"aligned"),
            ((4096, 8192), (1, 1 << 41), (0, 0), b"too large")):
        keep, a = args(ptrs, sizes, types)
        assert lib.dg_clip_grad_norm(*a, 2, 1.0, 256, 256, need, None) != 0
        assert text in lib.dg_last_error(), (text, lib.dg_last_error())
        assert lib.dg_grad_scale(*a, 256, None) != 0
        del keep
    keep, a = args((4096, 8192), (10, 10), (0, 0))
    for order, limit, norm, scratch, nbytes in ((3, 1.0, 256, 256, need), (-1, 1.0, 256, 256, need), (2, -1.0, 256, 256, need),
                                                (2, float("nan"), 256, 256, need), (2, 1.0, None, 256, need),
                                                (2, 1.0, 256, None, need), (2, 1.0, 256, 256, need - 1)):
        assert lib.dg_clip_grad_norm(*a, order, limit, norm, scratch, nbytes, None) != 0
    assert lib.dg_grad_scale(*a, None, None) != 0
    assert lib.dg_grad_norm(-1, None, None, None, 2, 1.0, 256, None, 256, need, None) != 0
    assert lib.dg_grad_norm(2, None, None, None, 2, 1.0, 256, None, 256, need, None) != 0


def test_shared_memory_is_found():
    """The comparison of gradients with gaps, against the sets of the bytes that they cover."""
    import itertools
    import random

    from dogs_amd import gradclip as G
    rng = random.Random(1)
    buffer = torch.zeros(400)

    def view():
        shape = [rng.randint(1, 5) for _ in range(rng.randint(1, 3))]
        strides = [rng.choice((0, 1, 2, 3, 4, 5, 7, 10, 12, 20)) for _ in shape]
        return buffer.view(rng.choice((torch.float32, torch.bfloat16))).as_strided(shape, strides, rng.randint(0, 40))

    def covered(t):
        e = t.element_size()
        return [t.data_ptr() + e * sum(i * s for i, s in zip(at, t.stride())) + b
                for at in itertools.product(*map(range, t.shape)) for b in range(e)]
    found = [0, 0]
    for _ in range(2000):
        views = [view() for _ in range(rng.randint(1, 4))]
        gapped = [k for k, t in enumerate(views) if not G._dense(t)]
        cover = [covered(t) for t in views]
        want = any(len(set(cover[k])) < len(cover[k]) for k in gapped) or any(
            set(cover[i]) & set(cover[j]) for i in range(len(views)) for j in range(i) if i in gapped or j in gapped)
        found[want] += 1
        if want:
            with pytest.raises(RuntimeError):
                G._check_apart(views, gapped, "clip")
        else:
            G._check_apart(views, gapped, "clip")
    assert min(found) > 100


def test_admm_run_refuses_clipping():
    """The ADMM rounds do not clip: a run that asks for it and has such rounds is refused before it trains anything."""
    from types import SimpleNamespace

    from dogs_amd.admm_run import ADMMRunConfig, block_train_config, pre_phase_iterations, run, run_sequential
    from dogs_amd.trainer import GSTrainConfig
    cfg = ADMMRunConfig(gs=GSTrainConfig(max_iterations=1000, densify_end_iter=300, max_grad_norm=0.1))
    start, pre = pre_phase_iterations(cfg), SimpleNamespace(spatial_lr_scale=5.0)
    assert 300 <= start < 1000
    for call in (lambda: run(cfg, None), lambda: run_sequential(cfg, [], "cuda:0"),
                 lambda: block_train_config(cfg, pre, start, 3)):
        with pytest.raises(ValueError, match="max_grad_norm"):
            call()
    cfg.gs.max_iterations = start                    # no round follows the pre-phase
    assert block_train_config(cfg, pre, start, 3).start_iteration == start
    cfg.gs.max_iterations, cfg.gs.max_grad_norm = 1000, 0.0
    cfg.gs.mask_max_grad_norm = 0.1                  # the rounds have no appearance mask
    assert block_train_config(cfg, pre, start, 3).sh_degree == 3


def test_appearance_batch_on_the_host():
    """The batched module on the CPU equals its single views; a view that is there twice adds both gradients."""
    from dogs_amd.masks import AppearanceEmbedding
    torch.manual_seed(0)
    net = AppearanceEmbedding(5).double()
    with torch.no_grad():
        net.appearance_embedding.normal_()
    images = torch.rand((3, 3, 2, 3), dtype=torch.float64)
    index = torch.tensor([4, 1, 4])
    masks = net(images, index, (33, 50))
    (masks ** 2).sum().backward()
    got = net.appearance_embedding.grad.clone()
    net.zero_grad()
    one = torch.stack([net(images[k], int(index[k]), (33, 50)) for k in range(3)])
    (one ** 2).sum().backward()
    assert torch.allclose(masks, one, rtol=1e-12, atol=1e-12)
    assert torch.allclose(got, net.appearance_embedding.grad, rtol=1e-9, atol=1e-12)
    with pytest.raises(ValueError):
        net(images, torch.tensor([4, 1]), (33, 50))
