"""Argument checks of the row operators (policy scores, 8-bit codes, products and checkpoints): everything here is
refused on the host, before anything reaches a GPU."""
import pytest
import torch

from muzero_amd import _hip

P = 0x1000   # a pointer no call below gets as far as using
F32, BF16 = _hip.TYPE_F32, _hip.TYPE_BF16


def _refused(rc, *words):
    assert rc < 0
    msg = _hip.lib().mz_last_error().decode()
    assert all(w in msg for w in words), msg


def test_policy_scores_refusals():
    f = _hip.lib().mz_policy_scores

    def call(logits=P, kind=F32, ld=8, actions=P, T=4, V=7, top=2, lp=P, ent=P, stats=P, ids=P, tlp=P):
        return f(logits, kind, ld, actions, T, V, top, lp, ent, stats, ids, tlp, None, 0, None)
    _refused(call(kind=9), "type")
    _refused(call(V=0), "V=0")
    _refused(call(T=-1), "T=-1")
    _refused(call(top=33, V=50, ld=50), "top=33")
    _refused(call(top=8), "top=8", "V=7")
    _refused(call(top=-1), "top=-1")
    _refused(call(ld=6), "stride")
    _refused(call(logits=None), "NULL")
    _refused(call(logits=P + 2), "misaligned")
    _refused(call(ent=None), "NULL")
    _refused(call(lp=None), "NULL")
    _refused(call(ids=None), "NULL")
    _refused(call(tlp=None), "NULL")
    assert call(T=0, logits=None, ent=None) == 0
    b = _hip.lib().mz_policy_scores_backward

    def back(logits=P, ld=7, actions=P, T=4, V=7, top=2, stats=P, ids=P, g=P, gh=P, gt=P, grad=P, ldg=7):
        return b(logits, F32, ld, actions, T, V, top, stats, ids, g, gh, gt, grad, ldg, None)
    _refused(back(grad=None), "NULL")
    _refused(back(ldg=5), "stride")
    _refused(back(stats=None), "NULL")
    _refused(back(ids=None), "NULL")
    _refused(back(actions=None), "NULL")
    assert back(T=0, logits=None, grad=None) == 0
    large = _hip.lib().mz_policy_scores_workspace(F32, 2, 200000, 32)
    if large:
        _refused(f(P, F32, 200000, P, 2, 200000, 32, P, P, P, P, P, None, 0, None), "workspace")
        _refused(f(P, F32, 200000, P, 2, 200000, 32, P, P, P, P, P, P, large - 1, None), "workspace")


def test_row_code_refusals():
    q, d = _hip.lib().mz_quant8_rows, _hip.lib().mz_dequant8_rows

    def quant(x=P, kind=F32, ldx=100, rows=4, K=100, bits=24, codes=P, ldc=128, scales=P):
        return q(x, kind, ldx, rows, K, bits, codes, ldc, scales, None)
    _refused(quant(kind=-1), "type")
    _refused(quant(K=0), "K=0")
    _refused(quant(K=(1 << 30) + 16, ldx=1 << 31, ldc=1 << 31), "K=")
    _refused(quant(rows=-1), "rows=-1")
    _refused(quant(ldx=99), "stride")
    _refused(quant(bits=8), "scale_bits")
    _refused(quant(x=None), "NULL")
    _refused(quant(codes=None), "NULL")
    _refused(quant(scales=None), "NULL")
    _refused(quant(ldc=96), "stride 96")
    _refused(quant(ldc=120), "stride 120")
    _refused(quant(codes=P + 8), "aligned")
    _refused(quant(x=P + 2), "misaligned")
    assert quant(rows=0, x=None, codes=None, scales=None) == 0
    _refused(d(P, 128, P, 4, 100, P, 7, 100, None), "type")
    _refused(d(P, 128, P, 4, 100, P, F32, 99, None), "stride")
    _refused(d(P, 128, None, 4, 100, P, F32, 100, None), "NULL")
    _refused(d(P, 96, P, 4, 100, P, F32, 100, None), "stride 96")


def test_int8_refusals():
    lib = _hip.lib()
    need = lib.mz_int8_workspace(4, 100, 50)
    assert need >= 4 * 128 + 16

    def fwd(x=P, kind=F32, ldx=100, rows=4, K=100, w=P, ldw=128, ws=P, N=50, act=0, y=P, ykind=F32, ldy=50, work=P, nwork=need):
        return lib.mz_int8_forward(x, kind, ldx, rows, K, w, ldw, ws, N, None, act, y, ykind, ldy, work, nwork, None)

    def coded(x=P, ldx=128, xs=P, rows=4, K=100, w=P, ldw=128, ws=P, N=50, act=0, y=P, ykind=F32, ldy=50):
        return lib.mz_int8_forward_codes(x, ldx, xs, rows, K, w, ldw, ws, N, None, act, y, ykind, ldy, P, 1 << 40, None)
    for f in (fwd, coded):
        _refused(f(rows=-1), "rows=-1")
        _refused(f(K=0), "K=0")
        _refused(f(N=0), "N=0")
        _refused(f(N=(1 << 26) + 1, ldy=1 << 27), "N=")
        _refused(f(w=None), "NULL")
        _refused(f(ws=None), "NULL")
        _refused(f(ldw=112), "128 bytes")
        _refused(f(w=P + 4), "aligned")
        _refused(f(act=4), "element-wise")
        _refused(f(ykind=5), "type")
        _refused(f(x=None), "NULL")
        _refused(f(y=None), "NULL")
        _refused(f(ldy=49), "stride 49")
        assert f(rows=0, x=None, y=None) == 0
    _refused(fwd(K=131073, ldx=131073, ldw=131200, nwork=1 << 40), "32-bit")
    _refused(coded(K=131073, ldx=131200, ldw=131200), "32-bit")
    _refused(fwd(kind=3), "type")
    _refused(fwd(ldx=99), "stride")
    _refused(fwd(work=None), "workspace")
    _refused(fwd(nwork=need - 1), "workspace")
    _refused(fwd(work=P + 8), "workspace")
    _refused(coded(xs=None), "NULL")
    _refused(coded(ldx=64), "128 bytes")


def test_checkpoint_refusals():
    lib = _hip.lib()
    RELU, TANH = _hip.ACT["relu"], _hip.ACT["tanh"]
    assert lib.mz_ckpt8_act_bytes(9, RELU) == 2 and lib.mz_ckpt8_act_bytes(9, TANH) == 9 and lib.mz_ckpt8_act_bytes(9, 0) == 0
    _refused(lib.mz_ckpt8_act_save(P, F32, 9, 4, 9, 0, P, None), "activation")
    _refused(lib.mz_ckpt8_act_save(P, F32, 9, 4, 9, RELU, None, None), "NULL")
    _refused(lib.mz_ckpt8_act_save(P, F32, 8, 4, 9, RELU, P, None), "stride")
    _refused(lib.mz_ckpt8_act_grad(P, F32, 9, None, 4, 9, RELU, P, 9, None), "NULL")
    _refused(lib.mz_ckpt8_act_grad(P, F32, 9, P, 4, 9, 4, P, 9, None), "activation")
    _refused(lib.mz_ckpt8_act_grad(P, F32, 9, P, 4, 9, RELU, None, 9, None), "NULL")
    need = lib.mz_ckpt8_workspace(F32, 3, 5000, 50, 100)
    assert need > 0 and lib.mz_ckpt8_workspace(F32, 3, 0, 50, 100) == 0 and lib.mz_ckpt8_workspace(F32, 3, 4, 50, 100) == 0

    def grad(dz=P, kind=F32, ldz=50, rows=5000, N=50, codes=P, ldc=128, scales=P, bits=3, K=100, dw=P, ldw=100, db=P, work=P, nwork=need):
        return lib.mz_ckpt8_weight_grad(dz, kind, ldz, rows, N, codes, ldc, scales, bits, K, dw, ldw, db, work, nwork, None)
    _refused(grad(rows=0), "rows=0")
    _refused(grad(rows=(1 << 20) + 1), "rows")
    _refused(grad(N=0), "N=0")
    _refused(grad(K=-1), "K=-1")
    _refused(grad(kind=3), "type")
    _refused(grad(bits=7), "scale_bits")
    for name in ("dz", "codes", "scales", "dw"):
        _refused(grad(**{name: None}), "NULL")
    _refused(grad(ldz=49), "stride")
    _refused(grad(ldw=99), "stride")
    _refused(grad(ldc=96), "stride")
    _refused(grad(dw=P + 2), "alignment")
    _refused(grad(work=None), "workspace")
    _refused(grad(nwork=need - 1), "workspace")


def test_python_refusals():
    from muzero_amd.checkpoints import checkpointed_linear, save_activations, weight_grad
    from muzero_amd.policy_scores import policy_scores
    from muzero_amd.quantized import QuantizedRows, int8_linear, quantize_rows
    z = torch.zeros(3, 5)
    for call in (lambda: policy_scores(z), lambda: quantize_rows(z), lambda: save_activations(z), lambda: checkpointed_linear(z, z)):
        with pytest.raises(_hip.HipError, match="GPU"):   # no CPU fallback
            call()
    for call in (lambda: policy_scores(z.double()), lambda: quantize_rows(z.long()), lambda: policy_scores([1.0]),
                 lambda: checkpointed_linear(z.double(), z)):
        with pytest.raises(TypeError):
            call()
    coded = QuantizedRows(torch.zeros(4, 128, dtype=torch.int8), torch.zeros(4), torch.Size((4, 100)), torch.float32, 24)
    rows = QuantizedRows(torch.zeros(2, 128, dtype=torch.int8), torch.zeros(2), torch.Size((2, 99)), torch.float32, 24)
    with pytest.raises(ValueError, match="99"):
        int8_linear(rows, coded)
    with pytest.raises(TypeError, match="QuantizedRows"):
        int8_linear(rows, torch.zeros(4, 99))
    rows = QuantizedRows(torch.zeros(2, 128, dtype=torch.int8), torch.zeros(2), torch.Size((2, 100)), torch.float32, 24)
    with pytest.raises(ValueError, match="activation"):
        int8_linear(rows, coded, activation="softmax")
    with pytest.raises(TypeError, match="out_dtype"):
        int8_linear(rows, coded, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="bias"):
        int8_linear(rows, coded, bias=torch.zeros(5))
    with pytest.raises(_hip.HipError, match="GPU"):
        weight_grad(torch.zeros(2, 3), rows)
    with pytest.raises(_hip.HipError, match="GPU"):   # codes on the CPU do not reach a kernel
        int8_linear(rows, coded)
    with pytest.raises(_hip.HipError, match="GPU"):
        rows.dequantize()


def test_rows_that_do_not_hold_their_shape_are_refused():
    """A kernel trusts the shape of QuantizedRows; whoever builds them by hand is checked."""
    from muzero_amd.quantized import QuantizedRows
    c, s = torch.zeros(4, 256, dtype=torch.int8), torch.zeros(4)
    make = lambda codes=c, scales=s, shape=(4, 200), dtype=torch.float32, bits=24: QuantizedRows(codes, scales, shape, dtype, bits)  # noqa: E731
    q = make()
    assert (q.rows, q.columns, q.ld, q.shape) == (4, 200, 256, torch.Size((4, 200))) and make(shape=(2, 2, 256)).rows == 4
    assert make(codes=torch.zeros(8, 256, dtype=torch.int8)[::2]).ld == 512
    for bad in (dict(codes=c.float()), dict(codes=c[0]), dict(scales=s.double()), dict(scales=torch.zeros(4, 1)), dict(dtype=torch.float64)):
        with pytest.raises(TypeError):
            make(**bad)
    for bad in (dict(shape=(4, 257)), dict(shape=(5, 200)), dict(shape=(4, 0)), dict(shape=()), dict(scales=torch.zeros(3)), dict(bits=8),
                dict(codes=c[:, :200]), dict(codes=c[:, ::2]), dict(codes=c[:, 8:136]), dict(codes=torch.zeros(4, 264, dtype=torch.int8)[:, :256]),
                dict(codes=c[:1].expand(4, 256)), dict(scales=torch.zeros(8)[::2])):
        with pytest.raises(ValueError):
            make(**bad)


def test_dense_sequences_are_recognised():
    from muzero_amd.checkpoints import eight_bit_checkpoints
    from muzero_amd.config import DenseLayerConfig, load_config
    from muzero_amd.neural_networks import DynamicsNetwork, PredictionNetwork
    from muzero_amd.neural_networks.network_builder import build_mlp, dense_pairs, is_dense_sequence
    seq, _ = build_mlp([DenseLayerConfig(out_features=8), DenseLayerConfig(out_features=3, activation="softmax")], 5)
    assert [a for _, a in dense_pairs(seq)] == ["relu", "softmax"]
    for bad in (torch.nn.Sequential(), torch.nn.Sequential(torch.nn.Linear(2, 2)), torch.nn.Sequential(torch.nn.Conv2d(1, 1, 1), torch.nn.ReLU())):
        assert not is_dense_sequence(bad)
        with pytest.raises(ValueError):
            dense_pairs(bad)
    cfg = load_config("config_c4_mlp.yaml")
    g = DynamicsNetwork(cfg.networks.latent_shape, 7, cfg.networks.dynamics)
    f = PredictionNetwork(cfg.networks.latent_shape, 7, cfg.networks.prediction)
    lat, act = torch.randn(3, *cfg.networks.latent_shape), torch.tensor([0, 3, 6])
    want = g(lat, act) + f(lat)
    with eight_bit_checkpoints(g, f) as outer:   # on the CPU the layers run as they are
        assert len(outer.sequences) == 3 and len(outer.merges) == 1
        with eight_bit_checkpoints(g, f):
            got = g(lat, act) + f(lat)
        assert "merge" in g.__dict__
    assert "merge" not in g.__dict__ and "forward" not in f.policy_mlp.__dict__
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    torch.testing.assert_close(torch.softmax(f.policy_logits(lat), 1), f(lat)[0])


def _small_networks():
    from muzero_amd.config import load_config
    from muzero_amd.neural_networks import DynamicsNetwork, PredictionNetwork
    cfg = load_config("config_c4_mlp.yaml")
    return (DynamicsNetwork(cfg.networks.latent_shape, 7, cfg.networks.dynamics),
            PredictionNetwork(cfg.networks.latent_shape, 7, cfg.networks.prediction), torch.randn(3, *cfg.networks.latent_shape))


def test_checkpoint_contexts_may_overlap_and_be_entered_again():
    from muzero_amd.checkpoints import eight_bit_checkpoints
    g, f, _ = _small_networks()
    a, b = eight_bit_checkpoints(g, f), eight_bit_checkpoints(g)
    a.__enter__(), b.__enter__()
    a.__exit__(None, None, None)                  # the first ends before the second
    assert "merge" in g.__dict__ and "forward" in g.reward_mlp.__dict__ and "forward" not in f.value_mlp.__dict__
    b.__exit__(None, None, None)
    assert "merge" not in g.__dict__ and "forward" not in g.reward_mlp.__dict__
    with a:
        with a:
            pass
        assert "merge" in g.__dict__
    assert "merge" not in g.__dict__
    with eight_bit_checkpoints(g, g):
        pass
    assert "merge" not in g.__dict__ and "forward" not in g.reward_mlp.__dict__


def test_copies_made_inside_a_context_are_themselves():
    import copy
    import io

    from muzero_amd.checkpoints import eight_bit_checkpoints
    g, f, lat = _small_networks()
    act = torch.tensor([0, 3, 6])
    with eight_bit_checkpoints(g, f):
        g2, f2 = copy.deepcopy(g), copy.deepcopy(f)
        data = io.BytesIO()
        torch.save((g, f), data)
    data.seek(0)
    g3, f3 = torch.load(data, weights_only=False)
    want = f(lat) + g(lat, act)
    with torch.no_grad():
        for p in list(g.parameters()) + list(f.parameters()):
            p.zero_()
    for gg, ff in ((g2, f2), (g3, f3)):
        assert all(torch.equal(x, y) for x, y in zip(want, ff(lat) + gg(lat, act)))
        with eight_bit_checkpoints(gg, ff) as ctx:
            assert len(ctx.sequences) == 3 and type(gg.__dict__["merge"]).__name__ == "_Taken"
        assert all(torch.equal(x, y) for x, y in zip(want, ff(lat) + gg(lat, act)))


def test_layers_that_do_more_than_a_layer_are_left_alone():
    from muzero_amd.checkpoints import eight_bit_checkpoints
    from muzero_amd.neural_networks.network_builder import is_dense_sequence

    class Twice(torch.nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    class Sum(torch.nn.Sequential):
        def forward(self, x):
            return super().forward(x) + x
    assert is_dense_sequence(torch.nn.Sequential(torch.nn.Linear(3, 3), torch.nn.ReLU()))
    assert not is_dense_sequence(torch.nn.Sequential(Twice(3, 3), torch.nn.ReLU()))
    assert not is_dense_sequence(Sum(torch.nn.Linear(3, 3), torch.nn.ReLU()))
    hooked = torch.nn.Sequential(torch.nn.Linear(3, 3), torch.nn.ReLU())
    hooked[0].register_forward_hook(lambda m, x, y: y + 1)
    assert not is_dense_sequence(hooked)
    own = torch.nn.Sequential(torch.nn.Linear(3, 3), torch.nn.ReLU())
    own.forward = lambda x: x
    with eight_bit_checkpoints(own):
        assert own(5) == 5
    assert own(5) == 5


@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_tangents_are_refused(grad_mode):
    """A result without a tangent would read as one that does not depend on the input: no call takes a dual tensor and
    drops its tangent, with reverse mode on or off."""
    import torch.autograd.forward_ad as fwad

    from muzero_amd.checkpoints import save_activations, weight_grad
    from muzero_amd.policy_scores import policy_scores
    from muzero_amd.quantized import QuantizedRows, int8_linear, quantize_rows
    z = torch.zeros(2, 100)
    coded = QuantizedRows(torch.zeros(4, 128, dtype=torch.int8), torch.zeros(4), torch.Size((4, 100)), torch.float32, 24)
    rows = QuantizedRows(torch.zeros(2, 128, dtype=torch.int8), torch.zeros(2), torch.Size((2, 100)), torch.float32, 24)
    with fwad.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = fwad.make_dual(z, torch.ones_like(z))
        bias = fwad.make_dual(torch.zeros(4), torch.ones(4))
        for call in (lambda: policy_scores(dual), lambda: policy_scores(dual[:, ::2]),
                     lambda: quantize_rows(dual), lambda: save_activations(dual), lambda: int8_linear(dual, coded),
                     lambda: weight_grad(dual, rows), lambda: int8_linear(rows, coded, bias)):
            with pytest.raises(NotImplementedError, match="tangent"):
                call()
        with pytest.raises(_hip.HipError, match="GPU"):   # a tensor without one is not refused for it
            policy_scores(z)
        with pytest.raises(_hip.HipError, match="GPU"):
            policy_scores(dual.detach())


def test_forward_mode_tangents_of_gradients_are_refused():
    import types

    import torch.autograd.forward_ad as fwad

    from muzero_amd.checkpoints import _CheckpointedLinear
    from muzero_amd.policy_scores import _gradient
    z = torch.zeros(2, 3)
    with fwad.dual_level():
        dy = fwad.make_dual(z, torch.ones_like(z))
        g = fwad.make_dual(torch.zeros(2), torch.ones(2))
        ctx = types.SimpleNamespace(saved_tensors=(z, None, torch.zeros(2, 3), None), kind=F32, needs_input_grad=(True,) * 4)
        for grads in ((g, None, None, None), (None, g, None, None), (None, None, None, dy)):
            with pytest.raises(NotImplementedError, match="tangent"):
                _gradient(ctx, *grads)
        ctx = types.SimpleNamespace(saved_tensors=(None, None, None, None), x_shape=(2, 5), needs_input_grad=(True,) * 4)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="tangent"):
            _CheckpointedLinear.backward(ctx, dy)


def test_a_context_ends_with_what_it_finds():
    """A forward that the user sets inside a context stays; an entry that is gone keeps nothing from being put back."""
    from muzero_amd.checkpoints import eight_bit_checkpoints
    g, f, lat = _small_networks()
    act = torch.tensor([0, 3, 6])
    want = g(lat, act) + f(lat)
    mine = lambda x: x + 1  # noqa: E731
    with eight_bit_checkpoints(g, f):
        f.value_mlp.forward = mine
    assert f.value_mlp.__dict__["forward"] is mine and f.value_mlp(1) == 2 and "forward" not in f.policy_mlp.__dict__
    del f.value_mlp.forward
    with eight_bit_checkpoints(g, f) as ctx:
        assert [t.name for t in ctx._open[0]].count("forward") == 3
        del ctx._open[0][0].module.forward             # the first of the list
        with eight_bit_checkpoints(f.value_mlp, g):    # takes it anew
            del g.merge
    nets = [m for net in (g, f) for m in net.modules()]
    assert all("forward" not in m.__dict__ and "merge" not in m.__dict__ for m in nets)
    outer, inner = eight_bit_checkpoints(f), eight_bit_checkpoints(f)
    outer.__enter__()
    f.policy_mlp.forward = mine
    inner.__enter__()                                  # leaves it alone
    outer.__exit__(None, None, None), inner.__exit__(None, None, None)
    assert f.policy_mlp.__dict__["forward"] is mine and "forward" not in f.value_mlp.__dict__
    del f.policy_mlp.forward
    assert all(torch.equal(x, y) for x, y in zip(want, g(lat, act) + f(lat)))


def test_a_forward_of_one_inner_layer_is_its_own():
    """Set on the instance, as a profiler or muzero_amd.neural_networks.per_call does it: on a Linear, an activation, the
    merge layer, the sequence itself."""
    from muzero_amd.checkpoints import eight_bit_checkpoints
    from muzero_amd.neural_networks.network_builder import dense_pairs, is_dense_sequence, is_plain
    from muzero_amd.quantized import Int8MLP
    for layer in (0, 1, None):
        seq = torch.nn.Sequential(torch.nn.Linear(3, 3), torch.nn.ReLU())
        m = seq if layer is None else seq[layer]
        m.forward = lambda x, f=m.forward: f(x) + 1
        assert not is_plain(m, type(m)) and not is_dense_sequence(seq)
        for refused in (lambda: dense_pairs(seq), lambda: Int8MLP(seq, device="cpu")):
            with pytest.raises(ValueError):
                refused()
        with eight_bit_checkpoints(seq) as ctx:
            assert ctx.sequences == []
        del m.forward
        m.forward = m.forward                          # the class's own method, bound: nothing of its own
        assert is_dense_sequence(seq) and len(eight_bit_checkpoints(seq).sequences) == 1
    g, f, lat = _small_networks()
    g.fc_merge.forward = lambda x: torch.nn.functional.linear(x, g.fc_merge.weight)
    act = torch.tensor([0, 3, 6])
    want = g(lat, act)
    with eight_bit_checkpoints(g) as ctx:
        assert ctx.merges == [] and all(torch.equal(x, y) for x, y in zip(want, g(lat, act)))
    with eight_bit_checkpoints(f), eight_bit_checkpoints(f) as ctx:   # what an open context put there is nobody's own
        assert len(ctx.sequences) == 2


def test_hooks_that_come_while_a_context_is_open(monkeypatch):
    """Such layers run as they are from then on, hooks and all, and go back to 8 bits when the hook has gone."""
    import muzero_amd.checkpoints as ck
    g, f, lat = _small_networks()
    act, kept = torch.tensor([0, 3, 6]), []

    def layer(x, weight, bias=None, activation="none"):
        kept.append(activation)
        return ck._activate_(torch.nn.functional.linear(x, weight, bias), activation)
    monkeypatch.setattr(ck, "checkpointed_linear", layer)
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    with ck.eight_bit_checkpoints(g, f):
        want = f(lat) + g(lat, act)
        assert len(kept) == 3 + 3 + 2 + 1
        seen = []
        hooks = [m.register_forward_hook(lambda m, x, y: (seen.append(m), y + 1)[1])
                 for m in (f.value_mlp[0], f.policy_mlp[1], g.fc_merge)]
        kept.clear()
        got = f(lat) + g(lat, act)
        assert seen == [f.value_mlp[0], f.policy_mlp[1], g.fc_merge]
        assert len(kept) == 2 and not any(torch.equal(x, y) for x, y in zip(want, got))
        for h in hooks:
            h.remove()
        every = torch.nn.modules.module.register_module_forward_hook(lambda m, x, y: seen.append(m))
        try:
            kept.clear(), seen.clear()
            f(lat)
            assert f.value_mlp[0] in seen and f.policy_mlp[4] in seen and not kept
        finally:
            every.remove()
        assert all(torch.equal(x, y) for x, y in zip(want, f(lat) + g(lat, act))) and len(kept) == 3 + 3 + 2 + 1


def test_autocast_keeps_no_copies_without_a_gradient(monkeypatch):
    """A layer that shares its weights with a checkpointed one in the same autocast region still has its gradient."""
    import muzero_amd.checkpoints as ck
    from muzero_amd.quantized import QuantizedRows
    monkeypatch.setattr(ck, "save_activations", lambda x: QuantizedRows(
        torch.zeros(x.shape[0], 128, dtype=torch.int8), torch.zeros(x.shape[0]), x.shape, x.dtype, 3))
    lin, x = torch.nn.Linear(4, 3), torch.randn(5, 4, requires_grad=True)
    with torch.autocast("cpu", torch.bfloat16):
        y = ck._CheckpointedLinear.apply(x, lin.weight, lin.bias, "none")
        z = lin(x)
    assert y.dtype == z.dtype == torch.bfloat16 and torch.equal(y, z)
    grads = torch.autograd.grad(z.sum(), (x, lin.weight, lin.bias))
    assert all(bool((g != 0).any()) for g in grads) and torch.is_autocast_cache_enabled()


def test_an_engine_shares_networks_of_the_precision_it_asks_for():
    import types

    from muzero_amd.quantized import Int8Networks
    from muzero_amd.selfplay import SelfPlayEngine

    class Reached(Exception):
        pass

    class Config:
        @property
        def mcts(self):
            raise Reached                              # the check is behind it
    eight, full = types.SimpleNamespace(nets=object.__new__(Int8Networks)), types.SimpleNamespace(nets=object())
    for share, int8 in ((eight, False), (full, True)):
        with pytest.raises(ValueError, match="int8"):
            SelfPlayEngine(None, None, None, 4, Config(), share=share, int8=int8)
    for share, int8 in ((eight, True), (full, False), (eight, None), (full, None), (None, True), (None, False)):
        with pytest.raises(Reached):
            SelfPlayEngine(None, None, None, 4, Config(), share=share, int8=int8)


def test_gradients_whose_sign_is_not_in_memory(monkeypatch):
    """A single value is contiguous whatever its stride, so the imaginary part of a conjugate reaches a kernel as a view
    with its minus sign left out.  What the kernel would read is read here."""
    import ctypes
    import types

    import muzero_amd.policy_scores as ps
    read = []

    class Lib:
        def mz_policy_scores_backward(self, *args):
            read.extend(ctypes.cast(p, ctypes.POINTER(ctypes.c_float))[0] for p in args[9:12])
            return 0
    monkeypatch.setattr(ps._hip, "lib", Lib)
    monkeypatch.setattr(ps, "stream_of", lambda t: 0)
    one = torch._neg_view(torch.tensor([2.5]))
    assert one.is_neg() and one.is_contiguous() and one.item() == -2.5
    ctx = types.SimpleNamespace(saved_tensors=(torch.zeros(1, 3), torch.zeros(1, dtype=torch.int64), torch.zeros(1, 3),
                                               torch.zeros(1, 1, dtype=torch.int64)), kind=F32)
    ps._gradient(ctx, one, one, None, one[:, None])
    assert read == [-2.5] * 3


def test_methods_inside_a_context_take_their_arguments_by_name():
    from muzero_amd.checkpoints import eight_bit_checkpoints
    g, f, lat = _small_networks()
    x, merged = lat.reshape(3, -1), torch.randn(3, g.fc_merge.in_features)
    want = f.value_mlp(input=x), g.merge(merged=merged)
    with eight_bit_checkpoints(g, f):
        assert torch.equal(f.value_mlp(input=x), want[0]) and torch.equal(g.merge(merged=merged), want[1])


def test_calls_of_more_rows_than_a_weight_gradient_takes_run_as_they_are(monkeypatch):
    import muzero_amd.checkpoints as ck
    seq, kept = torch.nn.Sequential(torch.nn.Linear(1, 1), torch.nn.Tanh()), []
    monkeypatch.setattr(ck, "checkpointed_linear", lambda x, *rest: (kept.append(len(x)), x)[1])
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    most = torch.zeros(1, 1).expand(ck.MAX_CHECKPOINT_ROWS + 1, 1)
    with ck.eight_bit_checkpoints(seq), torch.no_grad():
        assert seq(most).shape == most.shape and kept == []
        seq(most[1:])
    assert kept == [ck.MAX_CHECKPOINT_ROWS]


def test_scatter_rows_refusals():
    f = _hip.lib().mz_scatter_rows

    def call(x=P, ldx=8, rows=P, B=4, D=8, y=P, ldy=8):
        return f(x, ldx, rows, B, D, y, ldy, 10, None)
    _refused(call(B=-1), "rows=-1")
    _refused(call(D=0), "K=0")
    for name in ("x", "rows", "y"):
        _refused(call(**{name: None}), "NULL")
    _refused(call(ldx=7), "stride 7")
    _refused(call(ldy=7), "stride 7")
    _refused(call(y=P + 2), "misaligned")
    assert call(B=0, x=None, rows=None, y=None) == 0
