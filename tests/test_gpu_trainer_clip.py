"""GSTrainConfig.max_grad_norm and mask_max_grad_norm: the trainer's clipped steps.

* a limit that is never reached changes no bit (densification, reset and prune iterations included), whatever the route;
* a limit that is reached scales the first step's moments by the coefficient of the recorded norm;
* the appearance embedding's clipping gives the same bits on the native and the autograd route, and other ones than
  training without it."""
import copy
import math

import pytest
import torch

from test_gpu_trainer import _assert_same_state, _cfg, _normal, _problem, _route_state

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _run(dev, cfg, steps, native=False, net=None, seed=4):
    from dogs_amd.trainer import GaussianSplatTrainer
    m, cams, gts = _problem(dev, n_true=20_000, n_init=4_000, W=320, H=240, views=3)
    tr = GaussianSplatTrainer(m, cams, gts, cfg, device=dev, seed=seed, native=native, normal=_normal(dev, 5),
                              appear_embedding=copy.deepcopy(net))
    for _ in range(steps):
        tr.train_iteration()
    tr.sync()
    return tr


def test_a_limit_out_of_reach_changes_nothing(hip_device):
    kw = dict(densify_start_iter=2, densification_interval=4, opacity_reset_interval=7, prune_iterations=(10,),
              max_iterations=12)
    plain = _run(hip_device, _cfg(**kw), 12)
    clipped = _run(hip_device, _cfg(max_grad_norm=1e9, **kw), 12, native=True)
    assert {lg.route for lg in clipped.logs} == {"autograd"}
    assert any(lg.events for lg in clipped.logs)
    _assert_same_state(_route_state(plain), _route_state(clipped))
    assert plain.last_grad_norm is None and clipped.last_grad_norm.shape == ()


def test_the_recorded_norm_is_of_all_six_gradients(hip_device, monkeypatch):
    """Also in an iteration whose densification, reset or prune replaces tensors: not 0, and not of the rest alone."""
    from dogs_amd import trainer as T
    kw = dict(densify_start_iter=2, densification_interval=4, opacity_reset_interval=7, prune_iterations=(10,),
              max_iterations=12)
    tr = _run(hip_device, _cfg(max_grad_norm=1e9, **kw), 0)
    backward, want = torch.Tensor.backward, []

    def noting(self, *a, **k):
        backward(self, *a, **k)
        grads = [g["params"][0].grad for g in tr.optimizer.param_groups]
        want.append(math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads)))
    monkeypatch.setattr(T.torch.Tensor, "backward", noting)
    for _ in range(12):
        tr.train_iteration()
        assert abs(float(tr.last_grad_norm) - want[-1]) <= 2 * U * want[-1] and want[-1] > 0.0
    assert len(want) == 12
    assert {e for lg in tr.logs for e in lg.events} == {"densify", "reset_opacity", "prune"}


def test_a_limit_within_reach_scales_the_step(hip_device):
    kw = dict(densify_start_iter=10 ** 6, opacity_reset_interval=10 ** 6, prune_iterations=())
    free = _run(hip_device, _cfg(max_grad_norm=1e9, **kw), 1)
    norm = float(free.last_grad_norm)
    assert 0.0 < norm < math.inf
    limit = norm / 7
    tight = _run(hip_device, _cfg(max_grad_norm=limit, **kw), 1)
    assert float(tight.last_grad_norm) == norm
    c = limit / (norm + 1e-6)
    for a, b in zip(free.optimizer.param_groups, tight.optimizer.param_groups):
        name = a["name"]
        a, b = free.optimizer.state[a["params"][0]], tight.optimizer.state[b["params"][0]]
        # m = (1 - b1) g after the first step: each side rounds twice, the coefficient's norm and product twice more
        want = a["exp_avg"].double() * c
        assert bool(((b["exp_avg"].double() - want).abs() <= 8 * U * want.abs() + 2.0 ** -148).all())
        # SH degree 0 and equal scales: the higher colours and the rotations have no gradient in this step
        assert bool(b["exp_avg"].any()) == (name not in ("f_rest", "quaternion"))


def test_embedding_clipped_on_both_routes(hip_device):
    from dogs_amd.masks import AppearanceEmbedding
    torch.manual_seed(3)
    net = AppearanceEmbedding(3)
    with torch.no_grad():
        net.appearance_embedding.normal_(0.0, 0.3)
    kw = dict(densify_start_iter=10 ** 6, opacity_reset_interval=10 ** 6, prune_iterations=(), mask=True, lambda_mask=0.5)
    runs = [_run(hip_device, _cfg(mask_max_grad_norm=lim, **kw), 6, native=native, net=net)
            for native, lim in ((True, 1e-3), (False, 1e-3), (True, 0.0))]
    states = [{k: v.detach() for k, v in r.mask.state_dict().items()} for r in runs]
    assert {lg.route for lg in runs[0].logs} == {"native"}
    _assert_same_state(states[0], states[1])
    _assert_same_state(_route_state(runs[0]), _route_state(runs[1]))
    assert any(not torch.equal(states[0][k], states[2][k]) for k in states[0])
