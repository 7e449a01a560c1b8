"""The operators that train features, without a GPU: what they refuse, the shapes of
their torch.ops forms and the C entry points' status codes."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from dsl_splat_b200 import features, optim
from dsl_splat_b200._native import SplatAdamwTensor, lib

ops = torch.ops.splat200
P = 256  # an aligned address that is never read


def fake(*shape, dtype=torch.float32, device="cuda"):
    return torch.empty(shape, device=device, dtype=dtype)


@pytest.mark.parametrize("change, message", [
    (dict(activation="tanh"), "activation"),
    (dict(x=()), "x must have a last dimension"),
    (dict(x=(3, 0), weight=(0,)), "x must have a last dimension"),
    (dict(weight=(7,)), "weight must have shape"),
    (dict(bias=(1, 8)), "bias must have shape"),
    (dict(dtype=torch.float64), "x must be a CUDA"),
    (dict(weight_dtype=torch.float16), "weight must have x's dtype"),
    (dict(device="cpu"), "x must be a CUDA"),
    (dict(eps=0.0), "eps must be finite"),
    (dict(eps=1e-60), "eps must be finite"),
    (dict(x=(2, 65536), weight=(65536,), bias=(65536,)), "65535"),
])
def test_layer_norm_refusals(change, message):
    with FakeTensorMode():
        dtype, device = change.get("dtype", torch.float32), change.get("device", "cuda")
        x = fake(*change.get("x", (5, 8)), dtype=dtype, device=device)
        weight = fake(*change.get("weight", (8,)), dtype=change.get("weight_dtype", dtype),
                      device=device)
        bias = fake(*change.get("bias", (8,)), dtype=dtype, device=device)
        eps, act = change.get("eps", 1e-5), change.get("activation", "silu")
        for call in (lambda: features.layer_norm(x, weight, bias, eps=eps, activation=act),
                     lambda: ops.feature_layer_norm(x, weight, bias, eps, act),
                     lambda: ops.feature_layer_norm_backward(x, weight, bias, eps, act, x)):
            with pytest.raises(ValueError, match=message):
                call()


def test_layer_norm_refuses_host_tensors():
    with pytest.raises(ValueError, match="x must be a CUDA"):
        features.layer_norm(torch.zeros(2, 3))
    with FakeTensorMode(), pytest.raises(ValueError, match="upstream must have shape"):
        ops.feature_layer_norm_backward(fake(4, 8), None, None, 1e-5, "none", fake(4, 7))


@pytest.mark.parametrize("change, message", [
    (dict(table=(5,)), r"table must be \(V,C\)"),
    (dict(table=(0, 4)), r"table must be \(V,C\)"),
    (dict(table=(5, 0)), r"table must be \(V,C\)"),
    (dict(dtype=torch.float64), "table must be a CUDA"),
    (dict(device="cpu"), "table must be a CUDA"),
    (dict(ids_dtype=torch.int16), "ids must be an int32"),
    (dict(ids_device="cpu"), "ids must be on the table's device"),
    (dict(scale=float("nan")), "scale must be finite"),
    (dict(scale=1e39), "scale must be finite"),
    (dict(table=(5, 70000)), "65535"),
])
def test_embedding_refusals(change, message):
    with FakeTensorMode():
        table = fake(*change.get("table", (5, 4)), dtype=change.get("dtype", torch.float32),
                     device=change.get("device", "cuda"))
        ids = fake(3, 2, dtype=change.get("ids_dtype", torch.int64),
                   device=change.get("ids_device", "cuda"))
        scale = change.get("scale", 1.0)
        for call in (lambda: features.embedding(ids, table, scale=scale),
                     lambda: ops.feature_embedding(ids, table, scale)):
            with pytest.raises(ValueError, match=message):
                call()


def test_embedding_backward_refusals():
    with FakeTensorMode():
        ids = fake(3, 2, dtype=torch.int64)
        for upstream, entries, message in ((fake(3, 2), 5, "upstream must have the shape"),
                                           (fake(3, 3, 4), 5, "upstream must have the shape"),
                                           (fake(3, 2, 4), 0, r"table must be \(V,C\)")):
            with pytest.raises(ValueError, match=message):
                ops.feature_embedding_backward(ids, entries, 1.0, upstream)


def test_fake_shapes():
    with FakeTensorMode():
        x, w = fake(4, 5, 8, dtype=torch.bfloat16), fake(8, dtype=torch.bfloat16)
        assert features.layer_norm(x, w).shape == x.shape
        dx, dw, db = ops.feature_layer_norm_backward(x, w, None, 1e-5, "silu", x)
        assert dx.shape == x.shape and dw.shape == db.shape == (8,)
        ids, table = fake(3, 2, dtype=torch.int32), fake(9, 4, dtype=torch.float16)
        y = features.embedding(ids, table)
        assert y.shape == (3, 2, 4) and y.dtype is torch.float16
        assert ops.feature_embedding_backward(ids, 9, 1.0, y).shape == (9, 4)


@pytest.mark.parametrize("grad", [False, True])
def test_traced_programs_hold_the_operators(grad):
    def run(ids, table, w):
        return features.layer_norm(features.embedding(ids, table), w)

    with FakeTensorMode():
        tensors = [fake(*s).requires_grad_(grad) for s in ((9, 4), (4,))]
        graph = make_fx(run)(fake(6, dtype=torch.int64), *tensors)
    called = [n.target for n in graph.graph.nodes if n.op == "call_function"]
    assert ops.feature_embedding.default in called
    assert ops.feature_layer_norm.default in called


def test_forward_mode_is_refused():
    with FakeTensorMode(), fwAD.dual_level():
        x, table, ids = fake(6, 4), fake(9, 4), fake(3, dtype=torch.int64)
        for call in (lambda: features.layer_norm(fwAD.make_dual(x, torch.ones_like(x))),
                     lambda: features.embedding(ids, fwAD.make_dual(table, fake(9, 4))),
                     lambda: ops.feature_layer_norm(x, None, None, 1e-5, "none"),
                     lambda: ops.feature_embedding(ids, table, 1.0)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_decoder_takes_layer_norms():
    with FakeTensorMode():
        decoder = features.FeatureDecoder(features.Linear(fake(6, 4)),
                                          features.LayerNorm(fake(6), fake(6)))
        assert decoder(fake(2, 3, 4)).shape == (2, 3, 6)
        assert len(list(decoder.parameters())) == 3


def test_entry_points_refuse_before_any_launch():
    before = lib.splat_launch_count()
    norm, back = lib.splat_feature_layer_norm, lib.splat_feature_layer_norm_backward
    assert norm(3, 1, 8, P, None, None, 1e-5, 0, P, None) == -1
    assert norm(0, 1, 8, P, None, None, 1e-5, 5, P, None) == -1
    assert norm(0, 0, 8, P, None, None, 1e-5, 0, P, None) == -1
    assert norm(0, 1, 70000, P, None, None, 1e-5, 0, P, None) == -4
    assert norm(0, 1, 8, None, None, None, 1e-5, 0, P, None) == -1
    size = lib.splat_feature_layer_norm_backward_workspace_bytes
    assert size(0, 10, 8) >= 64 and size(4, 10, 8) == 0
    assert back(0, 10, 8, P, None, None, 1e-5, 0, P, P, P, P, P, 0, None) == -5
    assert back(0, 10, 8, P, None, None, 1e-5, 0, P, P, P, P, P + 4, 1 << 20, None) == -1
    assert back(0, 10, 8, P, None, None, 1e-5, 0, None, P, P, P, P, 1 << 20, None) == -1
    look, grad = lib.splat_feature_embedding, lib.splat_feature_embedding_backward
    assert look(0, 2, 1, 4, 4, P, P, 1.0, P, None) == -1
    assert look(0, 8, 0, 4, 4, P, P, 1.0, P, None) == -1
    assert look(0, 8, (1 << 30) + 1, 4, 4, P, P, 1.0, P, None) == -4
    assert look(0, 8, 1, 4, 4, None, P, 1.0, P, None) == -1
    assert lib.splat_feature_embedding_backward_workspace_bytes(0, 8, 4, 4) == 16
    assert lib.splat_feature_embedding_backward_workspace_bytes(0, 100000, 50, 4) > 400000
    assert grad(0, 8, 100000, 50, 4, P, P, 1.0, P, P, 100, None) == -5
    assert grad(0, 8, 8, 4, 4, P, P, 1.0, None, P, 100, None) == -1
    assert lib.splat_launch_count() == before


def test_embedding_gradients_of_common_entries_are_sorted():
    """No entry looks for more than 1024 rows of its own, however few entries there are."""
    size = lib.splat_feature_embedding_backward_workspace_bytes
    for dtype in range(3):
        for entries, channels in ((1, 1), (2, 512), (300, 32)):
            assert size(dtype, 1024, entries, channels) == 16
            assert size(dtype, 1025, entries, channels) > 16
    # nor are more steps than sorting takes spread over the device
    assert size(0, 64, 8192, 512) == 16 and size(0, 256, 8192, 512) > 16


def test_adamw_entry_points_refuse_before_any_launch():
    before = lib.splat_launch_count()

    def record(**change):
        values = dict(p=P, g=P, m=P, v=P, n=8, step=1, lr=0.1, beta1=0.9, beta2=0.999, eps=1e-8)
        return (SplatAdamwTensor * 1)(SplatAdamwTensor(**{**values, **change}))

    assert lib.splat_adamw(3, 32, 1, record(), 0, None) == -1
    assert lib.splat_adamw(0, 16, 1, record(), 0, None) == -1
    assert lib.splat_adamw(0, 32, -1, record(), 0, None) == -1
    assert lib.splat_adamw(0, 32, 1, None, 0, None) == -1
    assert lib.splat_adamw(0, 32, 1, record(step=0), 0, None) == -1
    assert lib.splat_adamw(0, 32, 1, record(p=None), 0, None) == -1
    assert lib.splat_adamw(0, 8, 1, record(), 0, None) == -1
    assert lib.splat_adamw(0, 32, 1, record(n=-1), 0, None) == -1
    assert lib.splat_adamw(0, 32, 1, record(n=1 << 41), 0, None) == -4
    assert lib.splat_adamw(0, 32, 0, None, 0, None) == 0
    assert lib.splat_adamw(0, 32, 1, record(n=0), 0, None) == 0
    assert lib.splat_adamw_decode(0, P, P, 0, P, None) == -1
    assert lib.splat_adamw_decode(8, None, P, 0, P, None) == -1
    assert lib.splat_adamw_encode(8, P, 0, P, None, None) == -1
    assert lib.splat_launch_count() == before


def test_optimizer_refuses_host_tensors_and_bad_settings():
    with pytest.raises(ValueError, match="CUDA"):
        optim.AdamW([torch.zeros(3, requires_grad=True)])
    with FakeTensorMode():
        p = fake(4, 3).requires_grad_()
        for change, message in ((dict(lr=-1.0), "lr"), (dict(lr=float("nan")), "lr"),
                                (dict(betas=(1.0, 0.9)), "betas"), (dict(eps=-1.0), "eps"),
                                (dict(weight_decay=-0.1), "weight_decay"),
                                (dict(state_bits=16), "state_bits")):
            with pytest.raises(ValueError, match=message):
                optim.AdamW([p], **change)
        with pytest.raises(ValueError, match="contiguous"):
            optim.AdamW([fake(4, 3).t().requires_grad_()])


def test_a_step_counted_on_the_host_is_not_captured(monkeypatch):
    """A replay would repeat its number."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with FakeTensorMode():
        p = fake(4, 3).requires_grad_()
        p.grad = fake(4, 3)
        optimizer = optim.AdamW([p], capturable=True)
        optimizer.state[p] = {"step": 3, "exp_avg": fake(4, 3), "exp_avg_sq": fake(4, 3)}
        with pytest.raises(RuntimeError, match="before a step is captured"):
            optimizer.step()
        with pytest.raises(ValueError, match="float32 tensors"):
            optimizer.set_moments(p, optim.Moment8(fake(4, 3, dtype=torch.uint8),
                                                   fake(1, dtype=torch.int8)), fake(4, 3))


@pytest.mark.parametrize("change, message", [
    (dict(eps=1e-50), "eps"), (dict(eps=1e-40), "eps"), (dict(eps=1e39), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(lr=1e39), "lr"),
    (dict(weight_decay=1e39), "weight_decay"), (dict(betas=(0.9, 1 - 2.0 ** -26)), "betas"),
])
def test_settings_that_float32_has_not(change, message):
    """They would become 0, infinity or 1 on the way to the kernel."""
    with FakeTensorMode():
        p = fake(4, 3).requires_grad_()
        with pytest.raises(ValueError, match=message):
            optim.AdamW([p], **change)
        settings = {"step": 1, "lr": 0.1, **change}
        with pytest.raises(ValueError, match=message):
            optim.adamw([p], [p], [p], [p], **settings)
        for eps in (0.0, 2.0 ** -126, 1e-15):
            optim.AdamW([p], eps=eps, betas=(0.0, 1 - 2.0 ** -24))


def test_moment8_refusals():
    codes, exponents = torch.zeros(300, dtype=torch.uint8), torch.zeros(2, dtype=torch.int8)
    optim.Moment8(codes, exponents)
    for c, e, message in ((codes.int(), exponents, "uint8"), (codes, exponents.int(), "int8"),
                          (codes, exponents[:1], "one value for each 256"),
                          (codes[::2], exponents[:1], "contiguous")):
        with pytest.raises(ValueError, match=message):
            optim.Moment8(c, e)
    with pytest.raises(ValueError, match="CUDA"):
        optim.Moment8(codes, exponents).values()
    with pytest.raises(ValueError, match="CUDA float32"):
        optim.Moment8.of(torch.zeros(3))


def torch_state(cls=torch.optim.AdamW, steps=3, dtype=torch.float32, **options):
    """A parameter and torch's state_dict of it after some steps."""
    p = torch.linspace(-1, 1, 12, dtype=dtype).reshape(4, 3).requires_grad_()
    optimizer = cls([p], **options)
    for step in range(steps):
        p.grad = torch.full_like(p, 0.5 + step)
        optimizer.step()
    return p, optimizer.state_dict()


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_loaded_states_of_torch(dtype, capturable):
    """torch counts its steps in float32 and holds moments in their parameter's type."""
    p, saved = torch_state(dtype=dtype)
    state = saved["state"][0]
    assert state["step"].dtype is torch.float32
    got = optim._loaded_state(state, p, 32, capturable)
    if capturable:
        assert got["step"].dtype is torch.int64 and got["step"].shape == ()
    else:
        assert type(got["step"]) is int
    assert int(got["step"]) == 3
    for name in ("exp_avg", "exp_avg_sq"):
        assert got[name].dtype is torch.float32 and got[name].is_contiguous()
        assert torch.equal(got[name], state[name].float())
        assert got[name].data_ptr() != state[name].data_ptr()
    # and this optimizer's own counts, of either kind
    for step in (3, torch.tensor(3)):
        assert int(optim._loaded_state({**state, "step": step}, p, 32, capturable)["step"]) == 3
    assert optim._loaded_state({}, p, 32, capturable) == {}


def test_loaded_states_that_are_refused():
    p, saved = torch_state(amsgrad=True)
    with pytest.raises(ValueError, match="amsgrad"):
        optim._loaded_state(saved["state"][0], p, 32, False)
    own = dict(state_bits=32)
    with pytest.raises(ValueError, match="amsgrad"):
        optim._check_loaded_group(saved["param_groups"][0], own)
    p, saved = torch_state()
    group, state = saved["param_groups"][0], saved["state"][0]
    optim._check_loaded_group(group, own)
    for change, message in ((dict(differentiable=True), "differentiable"),
                            (dict(decoupled_weight_decay=False), "decoupled"),
                            (dict(betas=(0.9, 1.0)), "betas"), (dict(state_bits=16), "state_bits")):
        with pytest.raises(ValueError, match=message):
            optim._check_loaded_group({**group, **change}, own)
    optim._check_loaded_group({**group, "decoupled_weight_decay": False, "weight_decay": 0.0}, own)
    for change, message in ((dict(step=torch.tensor(1.5)), "step"), (dict(step=-1), "step"),
                            (dict(step=torch.ones(2)), "step"), (dict(step=None), "step"),
                            (dict(step=torch.tensor(float("nan"))), "step"),
                            (dict(exp_avg=torch.zeros(3, 4)), "exp_avg must"),
                            (dict(exp_avg_sq=torch.zeros(4, 3, dtype=torch.uint8)), "exp_avg_sq"),
                            (dict(exp_avg=None), "exp_avg must")):
        with pytest.raises(ValueError, match=message):
            optim._loaded_state({**state, **change}, p, 32, False)


def test_steps_of_another_type_are_not_read(monkeypatch):
    """A state's counter on the device is read as 64-bit integers lie."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    with FakeTensorMode():
        for step in (fake(), fake(2, dtype=torch.int64), fake(dtype=torch.int64, device="cpu")):
            p = fake(4, 3).requires_grad_()
            p.grad = fake(4, 3)
            optimizer = optim.AdamW([p])
            optimizer.state[p] = {"step": step, "exp_avg": fake(4, 3), "exp_avg_sq": fake(4, 3)}
            with pytest.raises(ValueError, match="step must be"):
                optimizer.step()


ENTROPY = dict(x=(6, 4), weight=(9, 4), target=(6,), bias=(9,))


@pytest.mark.parametrize("change, message", [
    (dict(reduction="max"), "reduction"),
    (dict(x=()), "x must have a last dimension"),
    (dict(weight=(9,)), r"weight must be \(V,K\)"),
    (dict(weight=(0, 4), bias=(0,)), r"weight must be \(V,K\)"),
    (dict(weight=(9, 5)), "weight must have shape"),
    (dict(weight_dtype=torch.float16), "weight must have x's dtype"),
    (dict(bias=(8,)), "bias must have shape"),
    (dict(target=(5,)), "target must have x's device"),
    (dict(target=(6, 1)), "target must have x's device"),
    (dict(target_device="cpu"), "target must have x's device"),
    (dict(target_dtype=torch.uint8), "target must be an int32"),
    (dict(x_dtype=torch.float64), "x must be a CUDA"),
    (dict(ignore=1.5), "ignore_index"),
    (dict(ignore=True), "ignore_index"),
    (dict(ignore=1 << 63), "ignore_index"),
    (dict(weight=((1 << 20) + 1, 4), bias=((1 << 20) + 1,)), "2\\^20 words"),
])
def test_entropy_refusals(change, message):
    with FakeTensorMode():
        dtypes = dict(target=torch.int64)
        x, weight, target, bias = (
            fake(*change.get(m, ENTROPY[m]),
                 dtype=change.get(m + "_dtype", dtypes.get(m, torch.float32)),
                 device=change.get(m + "_device", "cuda")) for m in ENTROPY)
        with pytest.raises(ValueError, match=message):
            features.linear_cross_entropy(x, weight, target, bias,
                                          ignore_index=change.get("ignore", -100),
                                          reduction=change.get("reduction", "mean"))


def test_entropy_shapes_and_traces():
    with FakeTensorMode():
        x, w, b = (fake(*ENTROPY[m]).requires_grad_() for m in ("x", "weight", "bias"))
        target = fake(6, dtype=torch.int64)
        loss, moments, counted = ops.feature_entropy(x, w, target, b, -100, "none")
        assert loss.shape == (6,) and moments.shape == (6, 2) and counted.shape == (1,)
        dx, dw, db = ops.feature_entropy_backward(x, w, target, b, -100, "none", moments,
                                                  counted, loss)
        assert dx.shape == x.shape and dw.shape == w.shape and db.shape == b.shape
        with pytest.raises(ValueError, match="upstream must be float32 of shape"):
            ops.feature_entropy_backward(x, w, target, b, -100, "mean", moments, counted, loss)
        graph = make_fx(lambda x, w, t, b: features.linear_cross_entropy(x, w, t, b))(
            x, w, target, b)
        assert ops.feature_entropy.default in [n.target for n in graph.graph.nodes]
        image = fake(2, 3, 4)
        decoder = features.FeatureDecoder(features.LayerNorm(fake(4)), features.Linear(w, b))
        labels = fake(2, 3, dtype=torch.int64)
        assert decoder.cross_entropy(image, labels).shape == ()
        assert decoder.cross_entropy(image, labels, reduction="none").shape == (2, 3)
        for last in (features.Linear(w, b, "silu"), features.LayerNorm(fake(4))):
            with pytest.raises(ValueError, match="last Linear"):
                features.FeatureDecoder(features.Linear(fake(4, 4)), last).cross_entropy(image,
                                                                                        labels)


def test_entropy_entry_points_refuse_before_any_launch():
    before = lib.splat_launch_count()
    size = lib.splat_feature_entropy_workspace_bytes
    # only rows of several accumulators have their logits in memory
    assert size(0, 100, 513, 5000, 0) - size(0, 100, 512, 5000, 0) > 100 * 5000 * 4 - (1 << 17)
    assert size(0, 100, 0, 50, 0) == 0
    assert size(0, 100, 8, (1 << 20) + 1, 1) == 0

    def forward(dtype=0, rows=100, k=8, v=50, x=P, id_bytes=8, reduction=0, ws=P, n=1 << 30):
        return lib.splat_feature_entropy(dtype, rows, k, v, x, P, P, id_bytes, P, -100, reduction,
                                         P, None, None, ws, n, None)

    assert forward(dtype=5) == forward(rows=0) == forward(id_bytes=2) == forward(x=None) == -1
    assert forward(reduction=3) == forward(ws=P + 4) == -1
    assert forward(k=70000) == -4 and forward(n=100) == -5

    def backward(reduction=0, counted=P, bias=P, up=P, n=1 << 30):
        return lib.splat_feature_entropy_backward(0, 100, 8, 50, P, P, bias, 8, P, -100,
                                                  reduction, P, counted, up, P, P, P, P, n, None)

    assert backward(reduction=2, counted=None) == backward(bias=None) == backward(up=None) == -1
    assert backward(n=100) == -5
    assert lib.splat_launch_count() == before


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["random", "drawn", "largest"])
def test_the_bound_on_digits_tells_one_value_from_two(kind, dtype):
    """The bounds on the cross entropy's 16-bit gradients, on gradients in 64 bits whose dz alone
    is rounded: with upstreams of the rows' own one value of the type is refused and two pass;
    with a shared one, which is left to the results, one passes."""
    from test_entropy_gpu import ONE_VALUE, TWO_VALUES, digits, labels_of

    g = torch.Generator().manual_seed(37)
    x = torch.randn(2048, 64, generator=g).to(dtype)
    w = (torch.randn(512, 64, generator=g) / 2).to(dtype)
    target = labels_of(kind, x, w, 38)
    hit = torch.nn.functional.one_hot(target, 512).double()
    p_hit = torch.softmax(x.double() @ w.double().t(), 1) - hit

    def worst(up, within, values):
        dz = p_hit * up * within
        held = dz.to(dtype).double()
        if values == 2:
            held = held + (dz - held).to(dtype).double()
        held = held / within
        got = (held @ w.double()).to(dtype), (held.t() @ x.double()).to(dtype)
        return max(digits(x, w, target, "none", up.reshape(-1).float().expand(2048), got))

    scale = 2.0 ** 13 if dtype == torch.float16 else 0.25
    own = (1 + torch.randn(2048, generator=g).abs()).float().double()[:, None]
    assert worst(own, scale, 2) <= TWO_VALUES < worst(own, scale, 1)
    shared = torch.ones(1, 1, dtype=torch.float64)
    assert worst(shared, 4 * scale, 1) <= ONE_VALUE
