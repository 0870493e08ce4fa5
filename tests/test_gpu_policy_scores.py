"""policy_scores against the definition in 64 bits: values, alternatives, gradients, masked and empty rows, strides,
streams, replayed graphs, offsets past 32 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24                      # half a step of float32, relative
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}  # half a step below fp16's normal range
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _scores(*a, **k):
    from muzero_amd.policy_scores import policy_scores
    return policy_scores(*a, **k)


def _reference(logits, actions, top):
    """Everything in float64 on the CPU, plus the bounds of a float32 evaluation: d = z - m is rounded once (u |d|), an
    exponential and the terms of a sum of V numbers in any order of at least 16 parallel chains cost (V / 16 + 64) u of
    the sums of magnitudes."""
    z = logits.detach().cpu().to(torch.float64)
    T, V = z.shape
    m = z.max(1).values
    empty = torch.isneginf(m)
    d = z - torch.where(empty, torch.zeros_like(m), m)[:, None]
    e = torch.exp(d)
    S = e.sum(1)
    logS = torch.log(S)
    lp = d - logS[:, None]
    p = e / S[:, None]
    live = p > 0
    ed = torch.where(live, p * d, torch.zeros_like(p))           # p (z - m)
    ed2 = torch.where(live, p * d * d, torch.zeros_like(p))
    H = logS - ed.sum(1)
    n = V / 16 + 64
    err_logS = U * (n + ed.abs().sum(1) + logS.abs())
    err_lp = err_logS[:, None] + 2 * U * d.abs().clamp(max=1e30)
    err_H = err_logS + U * (n * (1 + ed.abs().sum(1)) + ed2.sum(1) + ed.abs().sum(1) ** 2)
    lp[empty], H[empty], p[empty] = -torch.inf, 0.0, 0.0
    err_H[empty] = 0.0
    ids = torch.sort(z + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
    return dict(lp=lp, H=H, p=p, err_lp=err_lp, err_H=err_H, ids=ids, empty=empty)


def _close(got, want, tol):
    got = got.detach().cpu().to(torch.float64)
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~(same | ((got - want).abs() <= tol))
    assert not bad.any(), (int(bad.sum()), got[bad][:5], want[bad][:5], torch.as_tensor(tol).expand_as(got)[bad][:5])


def _check(logits, actions, top, s=None):
    s = _scores(logits, actions, top=top) if s is None else s
    r = _reference(logits.reshape(-1, logits.shape[-1]), actions, top)
    _close(s.entropy.reshape(-1), r["H"], r["err_H"])
    if actions is not None:
        a = actions.cpu().long().reshape(-1, 1)
        none = a[:, 0] < 0
        a = a.clamp(min=0)
        want, tol = r["lp"].gather(1, a)[:, 0], r["err_lp"].gather(1, a)[:, 0]
        want[none], tol[none] = 0.0, 0.0
        _close(s.log_prob.reshape(-1), want, tol)
    if top:
        assert torch.equal(s.top_actions.reshape(-1, top).cpu(), r["ids"])
        _close(s.top_log_probs.reshape(-1, top), r["lp"].gather(1, r["ids"]), r["err_lp"].gather(1, r["ids"]))
    return s, r


def _make(T, V, dtype, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(T, V, generator=g) * spread * torch.rand(T, 1, generator=g)).to(dtype)
    return z.cuda(), torch.randint(0, V, (T,), generator=g).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,top", [(1, 1, 1), (1, 2, 2), (5, 7, 3), (4096, 7, 7), (3, 33, 32), (17, 64, 5), (9, 65, 32), (33, 255, 0),
                                     (6, 257, 8), (5, 1000, 20), (3, 1023, 1), (4, 1025, 32), (2, 4097, 16), (1, 8191, 32),
                                     (3, 32768, 5), (2, 50001, 32), (1, 131072, 20), (64, 20011, 3), (300, 2049, 4)])
def test_values_and_alternatives(T, V, top, dtype):
    z, a = _make(T, V, dtype, seed=T * 1000 + V)
    _check(z, a, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [7, 64, 300, 5000, 40000])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "masked", "lowest", "large", "one", "zeros"])
def test_hard_rows(V, kind, dtype):
    T, top = 5, min(V, 32)
    z, a = _make(T, V, dtype, seed=V)
    if kind == "equal":
        z = torch.full_like(z, 1.5)
    elif kind == "rising":  # every value larger than all before it
        z = torch.linspace(-20, 20, V, device="cuda").to(dtype).expand(T, V).contiguous()
    elif kind == "falling":
        z = torch.linspace(20, -20, V, device="cuda").to(dtype).expand(T, V).contiguous()
    elif kind == "masked":
        z[0] = -torch.inf                       # nothing left
        z[1, : V - 1] = -torch.inf              # one left, the last
        z[2, 1:] = -torch.inf                   # one left, the first
        z[3, ::2] = -torch.inf
    elif kind == "lowest":
        z[0] = torch.finfo(dtype).min
        z[1, : V // 2] = torch.finfo(dtype).min
        z[2, 1:] = torch.finfo(dtype).min
    elif kind == "large":
        z = z + 1000.0 if dtype != torch.float16 else z * 100
    elif kind == "one":
        z[:, V // 3] = 60.0
    elif kind == "zeros":  # 0 and -0 are equal
        z = torch.zeros_like(z)
        z[:, ::3] = -0.0
    _check(z, a, top)


@pytest.mark.parametrize("V", [7, 700, 30000])
def test_nan_and_infinity_are_loud(V):
    z, a = _make(4, V, torch.float32)
    z[0, V // 2] = torch.nan
    z[1, V - 1] = torch.inf
    z[2, :] = -torch.inf
    z[2, 0] = torch.nan
    top = 3
    s = _scores(z, a, top=top)
    assert s.log_prob[:3].isnan().all() and s.entropy[:3].isnan().all() and s.top_log_probs[:3].isnan().all()
    assert s.top_actions[0, 0] == V // 2 and s.top_actions[1, 0] == V - 1 and s.top_actions[2].tolist() == [0, 1, 2]
    _check(z[3:], a[3:], top, s._replace(log_prob=s.log_prob[3:], entropy=s.entropy[3:], top_actions=s.top_actions[3:],
                                         top_log_probs=s.top_log_probs[3:]))
    z.requires_grad_(True)
    s = _scores(z, a)
    s.log_prob.sum().backward()
    assert z.grad[:3].isnan().any(1).all() and not z.grad[3].isnan().any()


def test_actions_that_were_not_played_and_do_not_exist():
    z, a = _make(6, 50, torch.float32)
    a[1], a[2], a[3] = -1, 50, -100
    z.requires_grad_(True)
    s = _scores(z, a, top=1)
    assert s.log_prob[1] == 0 and s.log_prob[3] == 0 and s.log_prob[2].isnan() and s.entropy.isfinite().all()
    s.log_prob.sum().backward()
    assert (z.grad[[1, 3]] == 0).all() and z.grad[2].isnan().all() and z.grad[[0, 4, 5]].isfinite().all()


def _grad_reference(z64, actions, ids, g_lp, g_ent, g_top):
    """The formula in float64, and the bound of a float32 evaluation."""
    lp = torch.log_softmax(z64, 1)
    empty = torch.isneginf(z64).all(1)
    p = torch.exp(lp)
    plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    H = -plp.sum(1, keepdim=True)
    hot = torch.zeros_like(z64)
    mag = torch.zeros_like(z64)
    if g_lp is not None:
        hot.scatter_add_(1, actions[:, None], g_lp[:, None])
        mag.scatter_add_(1, actions[:, None], g_lp[:, None].abs())
    total = torch.zeros_like(H) if g_lp is None else g_lp[:, None].clone()
    size = total.abs()
    if g_top is not None:
        hot.scatter_add_(1, ids, g_top)
        mag.scatter_add_(1, ids, g_top.abs())
        total = total + g_top.sum(1, keepdim=True)
        size = size + g_top.abs().sum(1, keepdim=True)
    ge = torch.zeros_like(H) if g_ent is None else g_ent[:, None]
    grad = hot - p * total - ge * (plp + p * H)
    # log p is off by u (V / 16 + 64 + |log p| and what the entropy's bound holds), p by that relative to itself
    n = z64.shape[1] / 16 + 128 + lp.abs().clamp(max=200) * 4
    tol = U * (40 * mag + n * p * (size * 8 + ge.abs() * (lp.abs().clamp(max=200) + H + 1) * 8)) + 1e-37
    grad[empty], tol[empty] = 0.0, 0.0
    return grad, tol


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,top", [(1, 1, 0), (3, 2, 1), (1536, 7, 3), (5, 63, 0), (4, 130, 32), (7, 1024, 5), (3, 1025, 0), (2, 33333, 4),
                                     (64, 4099, 0)])
def test_gradient_matches_the_formula(T, V, top, dtype):
    z, a = _make(T, V, dtype, seed=V + 1)
    if V > 8:
        z[0, ::3] = -torch.inf
        z[T - 1] = -torch.inf
    z.requires_grad_(True)
    g = torch.Generator().manual_seed(5)
    g_lp, g_ent, g_top = (torch.randn(*s, generator=g, dtype=torch.float32).cuda() for s in ((T,), (T,), (T, top)))
    s = _scores(z, a, top=top)
    outs, gs = [s.log_prob, s.entropy], [g_lp, g_ent]
    if top:
        outs.append(s.top_log_probs), gs.append(g_top)
    # log p of a fully masked row is -inf: its incoming gradient must not matter
    got, = torch.autograd.grad(outs, z, gs)
    assert got.dtype == dtype and got.shape == z.shape
    d = lambda t: t.detach().cpu().double()  # noqa: E731
    want, tol = _grad_reference(d(z), a.cpu(), s.top_actions.cpu() if top else None, d(g_lp), d(g_ent),
                                d(g_top) if top else None)
    _close(got, want, tol + HALF[dtype] * (want.abs() + tol) + TINY[dtype])
    only_h, = torch.autograd.grad(_scores(z).entropy, z, g_ent)
    want, tol = _grad_reference(d(z), a.cpu(), None, None, d(g_ent), None)
    _close(only_h, want, tol + HALF[dtype] * (want.abs() + tol) + TINY[dtype])


def test_gradient_matches_differences():
    """Central differences of the float64 definition at h: error h^2 / 6 times a third derivative below 8 in size."""
    z, a = _make(3, 11, torch.float32, seed=3)
    z.requires_grad_(True)
    s = _scores(z, a, top=2)
    (s.log_prob.sum() * 0.7 - s.entropy.sum() * 0.3 + s.top_log_probs.sum() * 0.2).backward()
    z64, h = z.detach().cpu().double(), 1e-4

    def f(t):
        lp = torch.log_softmax(t, 1)
        return (lp.gather(1, a.cpu()[:, None]).sum() * 0.7 + (lp.exp() * lp).sum() * 0.3 + lp.gather(1, s.top_actions.cpu()).sum() * 0.2)
    for i in range(3):
        for j in range(11):
            e = torch.zeros_like(z64)
            e[i, j] = h
            diff = (f(z64 + e) - f(z64 - e)) / (2 * h)
            assert abs(float(z.grad[i, j]) - float(diff)) < 8 * h * h + 1e-6


@pytest.mark.parametrize("dtype", TYPES)
def test_shapes_strides_and_alignment(dtype):
    big, a = _make(24, 1300, dtype)
    for view in (big[:, :1001], big[:, 1:1002], big[::3, 5:905], big.t()[:1200].t(), big[:, ::2], big[3:4, 7:], big[:1].expand(24, 1300),
                 big.reshape(2, 3, 4, 1300), big[0]):
        V = view.shape[-1]
        act = torch.randint(0, V, view.shape[:-1], device="cuda", dtype=torch.int32)
        s, _ = _check(view, act, 4)
        assert s.log_prob.shape == view.shape[:-1] and s.top_actions.shape == view.shape[:-1] + (4,)
        leaf = view.detach().clone().requires_grad_(True)
        got, = torch.autograd.grad(_scores(leaf, act).log_prob.sum(), leaf)
        base = view.detach().as_strided(view.shape, view.stride(), view.storage_offset()).requires_grad_(True)
        got2, = torch.autograd.grad(_scores(base, act).log_prob.sum(), base)
        # the order of a row's sums follows its alignment, so the two agree with the formula and not bit for bit
        z64, a64 = view.detach().cpu().double().reshape(-1, V), act.cpu().long().reshape(-1)
        want, tol = _grad_reference(z64, a64, None, torch.ones(z64.shape[0], dtype=torch.float64), None, None)
        for g in (got, got2):
            _close(g.reshape(-1, V), want, tol + HALF[dtype] * (want.abs() + tol) + TINY[dtype])
    s = _scores(big[:0], a[:0], top=2)
    assert s.log_prob.shape == (0,) and s.top_actions.shape == (0, 2)
    z = big[:0].detach().requires_grad_(True)
    _scores(z, a[:0]).log_prob.sum().backward()
    assert z.grad.shape == (0, 1300)


def test_neighbours_are_left_alone():
    """A row's results do not depend on other rows, and nothing behind the last row is read into them."""
    z, a = _make(40, 3001, torch.float32)
    whole = _scores(z, a, top=9)
    z2 = z.clone()
    z2[20:] = torch.nan
    part = _scores(z2, a, top=9)
    for x, y in zip(whole, part):
        assert torch.equal(x[:20], y[:20])


def test_other_streams_and_replayed_graphs():
    z, a = _make(64, 50000, torch.bfloat16)
    z.requires_grad_(True)

    def step():
        s = _scores(z, a, top=6)
        g, = torch.autograd.grad((s.log_prob, s.entropy), z, (torch.ones_like(s.log_prob), torch.ones_like(s.entropy)))
        return s.log_prob.detach(), s.entropy.detach(), s.top_actions, s.top_log_probs.detach(), g
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    for turn in range(3):
        with torch.no_grad():
            z.copy_(torch.randn(64, 50000, generator=torch.Generator().manual_seed(turn)))
        want = step()
        for gr, out in zip(graphs, outs):
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(want, out)), turn


def test_offsets_past_32_bits():
    T, V = 70000, 32768  # 2.3e9 logits
    z = torch.zeros(T, V, dtype=torch.bfloat16, device="cuda")
    tail, a = _make(3, V, torch.bfloat16)
    z[-3:] = tail
    acts = torch.zeros(T, dtype=torch.int64, device="cuda")
    acts[-3:] = a
    s = _scores(z, acts, top=4)
    _check(tail, a, 4, s._replace(log_prob=s.log_prob[-3:], entropy=s.entropy[-3:], top_actions=s.top_actions[-3:],
                                  top_log_probs=s.top_log_probs[-3:]))
    assert (s.top_actions[:-3] == torch.arange(4, device="cuda")).all()
    z.requires_grad_(True)
    g, = torch.autograd.grad(_scores(z, acts).log_prob.sum(), z)
    small = tail.clone().requires_grad_(True)
    g2, = torch.autograd.grad(_scores(small, a).log_prob.sum(), small)
    assert torch.equal(g[-3:], g2)


def test_network_scores_and_learner_report():
    from muzero_amd.config import load_config
    from muzero_amd.neural_networks import PredictionNetwork
    from muzero_amd.policy_scores import score_actions
    cfg = load_config("config_c4_mlp.yaml")
    torch.manual_seed(0)
    f = PredictionNetwork(cfg.networks.latent_shape, 7, cfg.networks.prediction).cuda()
    lat = torch.randn(64, *cfg.networks.latent_shape, device="cuda")
    act = torch.arange(64, device="cuda") % 7
    s = score_actions(f, lat, act, top=7)
    policy, _ = f(lat)
    np.testing.assert_allclose(s.log_prob.exp().detach().cpu(), policy.gather(1, act[:, None])[:, 0].detach().cpu(), rtol=1e-5)
    assert torch.equal(s.top_actions[:, 0], policy.argmax(1))
    (-s.log_prob.mean() - 0.01 * s.entropy.mean()).backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for n, p in f.named_parameters() if n.startswith("policy"))


def test_results_may_be_changed_in_place_and_have_no_second_derivative():
    z, a = _make(5, 9, torch.float32)
    z.requires_grad_(True)
    s = _scores(z, a)
    assert s.top_actions is None and s.top_log_probs is None and _scores(z).log_prob is None
    want, = torch.autograd.grad(s.log_prob.clamp(min=-2.0).sum(), z)
    s = _scores(z, a)
    loss = s.log_prob.clamp_(min=-2.0).sum()
    s.entropy.detach().zero_()
    got, = torch.autograd.grad(loss, z)
    assert torch.equal(want, got)
    g, = torch.autograd.grad(_scores(z, a).entropy.sum(), z, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [65, 256, 257, 505, 513, 777, 1500, 1537, 2042, 2048, 2049, 3000, 3075, 4080, 4088, 4089, 4096])
@pytest.mark.parametrize("offset", [0, 3])
def test_row_lengths_between_the_variants(V, offset, dtype):
    """Every count of packs that a wave keeps, for rows on 16-byte addresses and off them, with more rows than one
    workgroup takes; the logits around a row hold larger values that no result may see."""
    g = torch.Generator().manual_seed(V)
    big = torch.full((13, V + 16 - V % 8), 500.0).to(dtype).cuda()
    z = big[:, offset : offset + V]
    z.copy_(torch.randn(13, V, generator=g).to(dtype))
    z[4] = -torch.inf
    z[5, 3:] = -torch.inf
    z[6, V - 1], z[7, 0] = 9.0, 9.0
    a = torch.randint(0, V, (13,), generator=g).cuda()
    _check(z, a, 8)
    _check(z, a, 0)
    base = z.detach().requires_grad_(True)  # keeps the strides and the offset
    g_lp, g_ent = (torch.randn(13, generator=g).cuda() for _ in range(2))
    s = _scores(base, a)
    got, = torch.autograd.grad([s.log_prob, s.entropy], base, [g_lp, g_ent])
    want, tol = _grad_reference(z.cpu().double(), a.cpu(), None, g_lp.cpu().double(), g_ent.cpu().double(), None)
    _close(got, want, tol + HALF[dtype] * (want.abs() + tol) + TINY[dtype])


def test_an_action_that_does_not_exist_spoils_only_its_own_score():
    z, a = _make(4, 30, torch.float32)
    a[1] = 30
    z.requires_grad_(True)
    s = _scores(z, a, top=2)
    got, = torch.autograd.grad(s.entropy.sum() + s.top_log_probs.sum(), z)
    t = _scores(z, None, top=2)
    want, = torch.autograd.grad(t.entropy.sum() + t.top_log_probs.sum(), z)
    assert s.log_prob[1].isnan() and got.isfinite().all() and torch.equal(got, want)


def test_views_with_a_pending_minus_sign():
    z, a = _make(5, 90, torch.float32)
    view = torch.conj(torch.complex(torch.zeros_like(z), z)).imag  # -z, not in memory yet
    assert view.is_neg()
    _check(view, a, 3, _scores(view, a, top=3))


def test_alternatives_out_of_range_are_not_written():
    """The C entry takes the list of alternatives from memory: an index outside the row changes nothing."""
    from muzero_amd import _hip
    z, a = _make(3, 40, torch.float32)
    stats = torch.tensor([[3.0, 2.0, 1.0]] * 3, device="cuda")
    ids = torch.tensor([[0, 40], [-1, 39], [1 << 40, 5]], device="cuda")
    g_top = torch.ones(3, 2, device="cuda")
    room = torch.full((5, 40), 7.0, device="cuda")
    p = _hip.ptr
    _hip.check(_hip.lib().mz_policy_scores_backward(p(z), _hip.TYPE_F32, 40, None, 3, 40, 2, p(stats), p(ids), None, None, p(g_top),
                                                    room[1:4].data_ptr(), 40, torch.cuda.current_stream().cuda_stream), "backward")
    assert (room[0] == 7).all() and (room[4] == 7).all() and room[1:4].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("T,V,top", [(1, 24577, 5), (3, 40000, 0), (2, 49153, 32), (96, 30011, 3), (95, 30011, 3), (256, 13001, 4),
                                     (257, 13001, 4), (300, 24000, 0), (97, 60000, 0)])
def test_long_rows_between_the_variants(T, V, top, dtype):
    z, a = _make(T, V, dtype, seed=T + V)
    z[0, :: 2] = -torch.inf
    z[T // 2] = 0.25                             # all equal
    z[T - 1, 1:] = torch.finfo(dtype).min
    _check(z, a, top)
