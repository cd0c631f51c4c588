"""Operators on a rank's state (tests/test_state_ops.py) where they meet what surrounds them:
checkpoints, other tensors than plain ones, transformations of a program."""
import pytest
import torch
import torch.distributed as dist

from state_oracles import keep_mask
from terraform_provider_iterative_amd import ops
from terraform_provider_iterative_amd.checkpoint import TrainingState


@pytest.mark.parametrize("consistent", [False, True])
def test_a_refusal_nobody_asked_for_does_not_keep_a_checkpoint_from_resuming(tmp_path, monkeypatch,
                                                                             consistent):
    """A device pool's refusal waits in its header for check(); a preemption may come before that."""
    def build():
        kv = torch.ones(10, 4)
        pool = ops.PagePool([kv], 4, 3, 4)
        return pool, TrainingState(torch.nn.Linear(2, 2), path=str(tmp_path / "spill"),
                                   tile_bytes=4096, paged={"kv": pool})

    pool, state = build()
    pool.extend([0, 1], [9, 3])
    books = pool.table.clone()
    with monkeypatch.context() as m:  # as on the device: no operation checks
        m.setattr(pool, "check", lambda: None)
        pool._header[1] = 1
        state.save({"step": 4})
    state.close()
    for _ in range(2):  # at the first start, and at every later one
        pool, state = build()
        with pytest.warns(UserWarning, match="not enough free pages"):
            if consistent:
                dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
                try:
                    meta = state.resume_consistent()
                finally:
                    dist.destroy_process_group()
            else:
                meta = state.resume()
        assert meta["step"] == 4 and state.step_value == 4
        assert torch.equal(pool.table, books) and pool.status()["error"] is None
        pool.extend([2], 1)
        state.close()


def test_the_books_of_another_pool_do_not_resume(tmp_path):
    def build(tokens):
        pool = ops.PagePool([torch.ones(10, 4)], tokens, 3, 4)
        return TrainingState(torch.nn.Linear(2, 2), path=str(tmp_path / "spill"), tile_bytes=4096,
                             paged={"kv": pool})

    state = build(4)
    state.save({"step": 4})
    state.close()
    state = build(2)
    with pytest.raises(ops.PageError, match="4 tokens a page"):
        state.resume()
    state.close()


def test_clearing_reaches_free_pages_that_a_copy_wrote():
    data = torch.ones(12, 4)
    pool = ops.PagePool([data], 4, 2, 12)
    pool.extend([0], 10)
    pool.compact(clear=True)
    pool.copy([0, 1], [9, 2])
    assert data[9].all()
    pool.copy([9], [7])
    pool.compact(clear=True)
    assert pool.refs.tolist() == [1] * 3 + [0] * 9
    assert data[:3].all() and not data[3:].any()


# -- tensors without memory of their own -----------------------------------------------------------

@pytest.fixture
def one_rank():
    dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    yield
    dist.destroy_process_group()


def _without_memory(kind):
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import Shard, distribute_tensor

    x = torch.ones(8, 4)
    if kind == "distributed":
        return distribute_tensor(x, init_device_mesh("cpu", (1,)), [Shard(0)])
    if kind == "fake":
        return FakeTensorMode().from_tensor(x)
    if kind in ("jagged", "nested"):
        layout = torch.jagged if kind == "jagged" else torch.strided
        return torch.nested.nested_tensor([x[:3], x[3:]], layout=layout)
    if kind in ("freed", "short"):
        x.untyped_storage().resize_(0 if kind == "freed" else 64)
        return x
    return {"sparse": x.to_sparse, "csr": x.to_sparse_csr, "mkldnn": x.to_mkldnn}[kind]()


@pytest.mark.parametrize("kind", ["distributed", "jagged", "nested", "freed", "short", "sparse",
                                  "csr", "mkldnn"])
def test_dropout_refuses_tensors_without_memory(kind, one_rank):
    refused = (TypeError, ValueError, RuntimeError)
    with pytest.raises(refused):
        ops.dropout(_without_memory(kind), 0.5, (1, 2))
    with pytest.raises(refused):
        ops.dropout(torch.ones(8, 4), 0.5, (1, 2), residual=_without_memory(kind))
    with pytest.raises(refused):
        ops.dropout(_without_memory(kind).requires_grad_(True), 0.5, (1, 2))


def test_dropout_refuses_a_state_without_memory():
    state = torch.zeros(2, dtype=torch.int64)
    state.untyped_storage().resize_(8)
    with pytest.raises(ValueError, match="memory of their own"):
        ops.dropout(torch.ones(8, 4), 0.5, ops.Draw(0, 0, state))


def test_dropout_of_a_distributed_tensors_local_part(one_rank):
    x = _without_memory("distributed")
    want = ops.dropout(torch.ones(8, 4), 0.5, (1, 2))
    assert torch.equal(ops.dropout(x.to_local(), 0.5, (1, 2), shard=((8, 4), (0, 0))), want)


@pytest.mark.parametrize("kind", ["distributed", "fake", "jagged", "nested", "freed", "short", "sparse",
                                  "csr", "mkldnn"])
def test_a_pool_refuses_tensors_without_memory(kind, one_rank):
    with pytest.raises((TypeError, ValueError, RuntimeError)):
        ops.PagePool([torch.ones(8, 4), _without_memory(kind)], 4, 2)


@pytest.mark.parametrize("kind", ["distributed", "fake", "freed"])
def test_a_pool_refuses_numbers_without_memory(kind, one_rank):
    pool = ops.PagePool([torch.ones(8, 4)], 4, 2)
    slots = torch.zeros(1, dtype=torch.int64)
    if kind == "freed":
        slots.untyped_storage().resize_(0)
    else:
        slots = _without_memory(kind).to(torch.int64).flatten()[:1]
    before = pool.meta.clone()
    for call in (lambda: pool.extend(slots, 1), lambda: pool.extend([0], slots),
                 lambda: pool.fork(slots, [1]), lambda: pool.free(slots),
                 lambda: pool.copy(slots, [2]), lambda: pool.copy([2], slots)):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            call()
    assert torch.equal(pool.meta, before)


# -- transformations of a program ------------------------------------------------------------------

KEY = ((1 << 64) - 3, 7)  # a seed that has no sign


def _block(x):
    return ops.dropout(x * 2, 0.4, KEY, residual=x) + 1


def _block_gradient(x):
    x = x.detach().requires_grad_(True)
    return torch.autograd.grad(_block(x).sum(), x)[0]


def _live_state(x):
    x = x.detach().requires_grad_(True)
    y = ops.dropout(x, 0.4, ops.Draw(0, 2, STATE))
    return torch.autograd.grad(y.sum(), x)[0]


STATE = torch.tensor([5, 6])


@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
@pytest.mark.parametrize("f", [_block, _block_gradient])
def test_a_graph_of_dropout_computes_dropout(f, mode):
    from torch.fx.experimental.proxy_tensor import make_fx

    traced = make_fx(f, tracing_mode=mode)(torch.randn(6, 11))
    x = torch.randn(6, 11)
    assert torch.equal(traced(x), f(x))


def test_a_graph_of_a_draw_with_a_state():
    from torch.fx.experimental.proxy_tensor import make_fx

    traced, x = make_fx(_live_state)(torch.randn(40)), torch.randn(40)
    assert torch.equal(traced(x), ops.dropout(torch.ones(40), 0.4, (5, 8)))


def test_a_traced_and_an_exported_program_compute_dropout():
    traced = torch.jit.trace(_block, (torch.randn(6, 11),))
    x = torch.randn(6, 11)
    assert torch.equal(traced(x), _block(x))

    class Net(torch.nn.Module):
        def forward(self, x):
            return _block(x)

    assert torch.equal(torch.export.export(Net(), (x,)).module()(x), _block(x))


@pytest.mark.parametrize("dtype,residual", [(torch.bfloat16, None), (torch.bfloat16, torch.float32),
                                            (torch.float16, torch.float16)])
def test_dropout_of_fake_tensors(dtype, residual):
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode

    with FakeTensorMode():
        x = torch.ones(5, 7, dtype=dtype).t().requires_grad_(True)
        r = None if residual is None else torch.ones(7, 5, dtype=residual)
        out = ops.dropout(x, 0.5, (1, 2), residual=r)
        grad, = torch.autograd.grad(out.sum(), x)
    assert type(out) is type(grad) is FakeTensor
    assert out.shape == grad.shape == (7, 5) and grad.dtype == dtype
    assert out.dtype == (residual or dtype) and out.stride() == ((1, 7) if r is None else (5, 1))


def test_a_stream_is_refused_in_a_trace():
    from torch.fx.experimental.proxy_tensor import make_fx

    masks, x = ops.MaskStream(3), torch.ones(8)
    for trace in (torch.jit.trace, lambda f, args: make_fx(f)(*args)):
        with pytest.raises(ValueError, match="traced"):
            trace(lambda v: ops.dropout(v, 0.5, masks), (x,))
    assert masks.number == 0
    compiled = torch.compile(lambda v: ops.dropout(v, 0.5, masks) * 2, backend="eager")
    for number in range(3):
        assert torch.equal(compiled(x), ops.dropout(x, 0.5, (3, number)) * 2)
    assert masks.number == 3


def test_the_operators_own_refusals():
    """A traced program may be given other tensors than it was traced with."""
    x = torch.ones(4, 4)
    good = dict(x=x, residual=None, dtype=torch.float32, threshold=1 << 31, scale=2.0, seed=1, number=2,
                state=None, first=0, strides=[])
    assert torch.equal(torch.ops.tpi.dropout(**good), ops.dropout(x, 0.5, (1, 2)))
    for bad in (dict(x=x.double()), dict(dtype=torch.float64), dict(dtype=torch.int16),
                dict(x=x.half(), dtype=torch.bfloat16), dict(residual=x.half()),
                dict(residual=x.half(), dtype=torch.float16),
                dict(residual=torch.ones(4)), dict(threshold=-1), dict(threshold=(1 << 32) + 1),
                dict(number=-1), dict(first=-1), dict(strides=[1]), dict(state=torch.zeros(2)),
                dict(state=torch.zeros(3, dtype=torch.int64)),
                dict(used=torch.zeros(1, dtype=torch.int64)), dict(x=x.to_sparse())):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            torch.ops.tpi.dropout(**{**good, **bad})


@pytest.mark.parametrize("dtype,kind", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                        (torch.float16, torch.float16)])
@pytest.mark.parametrize("which", ["x", "residual", "both"])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_carries_the_tangents(dtype, kind, which, requires_grad):
    """The operator is linear: its tangent is itself, of x's tangent, plus the residual's."""
    import torch.autograd.forward_ad as forward

    g = torch.Generator().manual_seed(5)
    x, tx = (torch.randn(9, 21, generator=g).to(dtype) for _ in range(2))
    r, tr = (torch.randn(9, 21, generator=g).to(kind) for _ in range(2))
    with forward.dual_level():
        a = x.clone().requires_grad_(requires_grad)
        b = r.clone().requires_grad_(requires_grad)
        out = ops.dropout(a if which == "residual" else forward.make_dual(a, tx), 0.4, KEY,
                          residual=b if which == "x" else forward.make_dual(b, tr))
        primal, tangent = forward.unpack_dual(out)
        assert torch.equal(primal, ops.dropout(x, 0.4, KEY, residual=r))
        want = {"x": lambda: ops.dropout(tx, 0.4, KEY, residual=torch.zeros_like(r)),
                "residual": lambda: tr, "both": lambda: ops.dropout(tx, 0.4, KEY, residual=tr)}
        assert tangent.dtype == kind and torch.equal(tangent, want[which]())
        if requires_grad:
            grads = torch.autograd.grad(primal.sum(), (a, b))
            assert torch.equal(grads[0], ops.dropout(torch.ones_like(x), 0.4, KEY))
            assert torch.equal(grads[1], torch.ones_like(r))
    alone = torch.func.jvp(lambda v: ops.dropout(v, 0.4, KEY), (x,), (tx,))[1]
    assert torch.equal(alone, ops.dropout(tx, 0.4, KEY))


def test_forward_mode_of_a_state_and_over_the_reverse():
    import torch.autograd.forward_ad as forward

    x, tx, w = (torch.randn(30, generator=torch.Generator().manual_seed(i)) for i in range(3))
    with forward.dual_level():
        v = forward.make_dual(x.clone().requires_grad_(True), tx)
        out = ops.dropout(v, 0.4, ops.Draw(0, 2, STATE))
        assert torch.equal(forward.unpack_dual(out).tangent, ops.dropout(tx, 0.4, (5, 8)))
        # d/dt of the gradient of sum(w out^2): the operator, applied to 2 w times the tangent
        gradient, = torch.autograd.grad((w * out ** 2).sum(), v, create_graph=True)
        want = ops.dropout(2 * w * ops.dropout(tx, 0.4, (5, 8)), 0.4, (5, 8))
        assert torch.allclose(forward.unpack_dual(gradient).tangent, want)
    torch.autograd.gradcheck(lambda a, b: ops.dropout(a, 0.4, KEY, residual=b).double(),
                             (torch.ones(11, requires_grad=True), torch.ones(11, requires_grad=True)),
                             eps=0.25, atol=1e-5, check_forward_ad=True)


# -- gradients and tangents of layouts that the caller did not choose ------------------------------

def _turned(t):
    """The same values, no two dimensions of which can be walked as one."""
    order = list(range(t.dim()))[::-1]
    return t.permute(order).contiguous().permute(order)


@pytest.mark.parametrize("shard", [None, ((2,) * 6 + (5,), (0,) * 6 + (1,))])
def test_a_gradient_of_many_dimensions_in_any_layout(shard):
    x = torch.randn([2] * 6 + [3], requires_grad=True)
    out = ops.dropout(x, 0.4, KEY, shard=shard)
    grad = torch.randn(x.shape)
    assert _turned(grad).stride() != grad.stride()
    want = ops.dropout(grad, 0.4, KEY, shard=shard)
    dx, = torch.autograd.grad(out, x, _turned(grad).requires_grad_(True), create_graph=True)
    assert torch.equal(dx, want)


def test_a_tangent_of_many_dimensions_in_any_layout():
    x, t, r = (torch.randn([2] * 7) for _ in range(3))
    got = torch.func.jvp(lambda a, b: ops.dropout(a, 0.4, KEY, residual=b), (x, r),
                         (_turned(t), _turned(t) * 2))[1]
    assert torch.equal(got, ops.dropout(t, 0.4, KEY, residual=t * 2))


@pytest.mark.parametrize("dtype,kind", [(torch.float32, None), (torch.bfloat16, torch.float32)])
def test_a_gradient_without_storage_is_a_zero_one(dtype, kind):
    x = torch.randn(6, 5).to(dtype).requires_grad_(True)
    r = None if kind is None else torch.randn(6, 5).to(kind).requires_grad_(True)
    out = ops.dropout(x, 0.4, KEY, residual=r)
    zero = torch._efficientzerotensor((6, 5), dtype=out.dtype)
    grads = torch.autograd.grad(out, (x,) if r is None else (x, r), zero)
    for grad, of in zip(grads, (x, r)):
        assert grad.dtype == of.dtype and grad.shape == of.shape and not grad.any()


# -- blocks that are computed twice ----------------------------------------------------------------

def test_a_device_streams_draw_keeps_its_mask():
    masks, x = ops.MaskStream(3, device="cpu"), torch.ones(300)
    first, second = masks.next(), masks.next()
    masks.advance()
    third = masks.next()
    masks.advance()
    masks.load_state_dict({"seed": 9, "number": 5})
    fourth = masks.next()
    for draw, key in ((first, (3, 0)), (second, (3, 1)), (third, (3, 2)), (fourth, (9, 5)),
                      (first, (3, 0))):
        assert torch.equal(ops.dropout(x, 0.5, draw), ops.dropout(x, 0.5, key))
    assert masks.state_dict() == {"seed": 9, "number": 6}


def test_a_device_streams_draws_do_not_come_from_a_trace():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    masks, x = ops.MaskStream(3, device="cpu"), torch.ones(300)
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        ops.dropout(mode.from_tensor(x), 0.5, masks)
    graph = make_fx(lambda v: ops.dropout(v, 0.5, masks))(x)  # draw 1 of whatever the step begins with
    assert torch.equal(ops.dropout(x, 0.5, masks), ops.dropout(x, 0.5, (3, 2)))
    assert torch.equal(graph(x), ops.dropout(x, 0.5, (3, 1)))
    masks.advance()
    assert torch.equal(graph(x), ops.dropout(x, 0.5, (3, 4)))


@pytest.mark.parametrize("device", [None, "cpu"])
@pytest.mark.parametrize("reentrant", [False, True])
def test_a_block_computed_twice_with_a_draw_from_outside(device, reentrant):
    from torch.utils.checkpoint import checkpoint

    masks = ops.MaskStream(3, device=device)
    torch.manual_seed(0)
    a, b = torch.nn.Linear(32, 48), torch.nn.Linear(48, 8)
    x = torch.randn(16, 32, requires_grad=True)

    def gradients(draw, twice):
        def block(v):
            return b(ops.dropout(a(v), 0.5, draw))
        y = checkpoint(block, x, use_reentrant=reentrant) if twice else block(x)
        if masks.state is not None:
            masks.advance()  # before the backward pass
        return torch.autograd.grad(y.pow(2).sum(), [x, *a.parameters(), *b.parameters()]) \
            if not reentrant else _backward(y, [x, *a.parameters(), *b.parameters()])

    def _backward(y, inputs):
        for p in inputs:
            p.grad = None
        y.pow(2).sum().backward()
        return [p.grad for p in inputs]

    for number in range(3):
        got, want = gradients(masks.next(), True), gradients((3, number), False)
        assert all(torch.equal(g, w) for g, w in zip(got, want))


class _Blocks(torch.nn.Module):
    """Linear, CounterDropout, Linear, twice: the second block inside the first one's last layer."""

    def __init__(self, masks):
        super().__init__()
        torch.manual_seed(0)
        self.masks = masks
        self.a, self.b, self.c, self.d = (torch.nn.Linear(24, 24) for _ in range(4))
        self.one, self.two = ops.CounterDropout(0.5, masks), ops.CounterDropout(0.3, masks)

    def inner(self, x):
        return self.d(self.two(self.c(x)))

    def outer(self, x, inner):
        x = self.b(self.one(self.a(x), x))
        return inner(x) + self.two(x)

    def gradients(self, x, checkpoint, nested=False, times=1):
        inner = (lambda v: checkpoint(self.inner, v)) if nested else self.inner
        y = checkpoint(lambda v: self.outer(v, inner), x).pow(2).sum()
        if self.masks.state is not None:
            self.masks.advance()
        for i in range(times):
            out = torch.autograd.grad(y, [x, *self.parameters()], retain_graph=i + 1 < times)
        return out


@pytest.mark.parametrize("device", [None, "cpu"])
@pytest.mark.parametrize("nested", [False, True])
@pytest.mark.parametrize("compiled", [False, True])
def test_checkpointed_layers_draw_the_same_masks_twice(device, nested, compiled):
    from torch.utils.checkpoint import checkpoint

    if compiled:
        torch._dynamo.reset()
    once, twice = (_Blocks(ops.MaskStream(3, device=device)) for _ in range(2))
    x = torch.randn(16, 24, requires_grad=True)
    if compiled:
        twice.outer = torch.compile(twice.outer, backend="eager")
    for step in range(3):
        want = once.gradients(x, lambda f, v: f(v))
        got = twice.gradients(x, lambda f, v: checkpoint(
            f, v, use_reentrant=False, context_fn=twice.masks.checkpoint_contexts), nested, 1 + step)
        assert all(torch.equal(g, w) for g, w in zip(got, want))
        assert twice.masks.state_dict() == once.masks.state_dict() == {"seed": 3, "number": 3 * step + 3}


@pytest.mark.parametrize("device", [None, "cpu"])
@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("compiled", [False, True])
def test_a_second_computation_without_the_contexts_is_refused(device, reentrant, compiled):
    from torch.utils.checkpoint import checkpoint

    masks = ops.MaskStream(3, device=device)
    block = torch.nn.Sequential(torch.nn.Linear(24, 24), ops.CounterDropout(0.5, masks),
                                torch.nn.Linear(24, 24))
    run = torch.compile(block, backend="eager") if compiled else block
    y = checkpoint(run, torch.randn(4, 24, requires_grad=True), use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="computes again"):
        y.sum().backward()
    assert masks.state_dict()["number"] == 1
    block(torch.randn(4, 24)).sum().backward()  # and the stream goes on
    assert masks.state_dict()["number"] == 2


def test_a_checkpointed_layer_with_a_draw():
    from torch.utils.checkpoint import checkpoint

    masks = ops.MaskStream(3)
    layer, x = ops.CounterDropout(0.5, masks), torch.randn(40, requires_grad=True)
    draw = masks.next()
    y = checkpoint(lambda v: layer(v, draw=draw).pow(2), x, use_reentrant=True)
    y.sum().backward()
    dropped = ops.dropout(x.detach(), 0.5, (3, 0))
    assert torch.equal(x.grad, ops.dropout(2 * dropped, 0.5, (3, 0))) and masks.number == 1
    layer.eval()
    assert layer(x, draw=draw) is x


def test_a_block_that_draws_more_the_second_time_is_refused():
    from torch.utils.checkpoint import checkpoint

    masks, count = ops.MaskStream(3), []

    def block(v):
        count.append(0)
        for _ in count:
            v = ops.dropout(v, 0.5, masks)
        return v.pow(2)

    y = checkpoint(block, torch.ones(8, requires_grad=True), use_reentrant=False,
                   context_fn=masks.checkpoint_contexts)
    with pytest.raises(RuntimeError, match="draws more masks"):
        y.sum().backward()
    assert masks.number == 1


def test_a_model_with_its_stream_can_be_copied_and_pickled():
    import copy
    import pickle

    for device in (None, "cpu"):
        model = _Blocks(ops.MaskStream(3, device=device))
        model.one(torch.ones(8))
        for other in (copy.deepcopy(model), pickle.loads(pickle.dumps(model))):
            assert other.one.stream is other.masks is not model.masks
            assert torch.equal(other.one(torch.ones(8)), ops.dropout(torch.ones(8), 0.5, (3, 1)))
        assert model.masks.state_dict()["number"] == 1


# -- builds ----------------------------------------------------------------------------------------

def test_the_host_operators_build_without_rocm(tmp_path, monkeypatch):
    """With a torch that is not built for ROCm, and no ROCm there, _tpi_torch serves host tensors."""
    import os
    import subprocess
    import sys

    from terraform_provider_iterative_amd import _build

    target = str(tmp_path / os.path.basename(_build.TORCH_EXT))
    monkeypatch.setattr(torch.version, "hip", None)
    monkeypatch.setattr(_build, "TORCH_EXT", target)
    monkeypatch.setattr(_build, "LIB", str(tmp_path))
    monkeypatch.setattr(_build, "ROCM_LIB", str(tmp_path / "rocm" / "lib"))
    assert _build.build_torch_ext() == target
    needed = subprocess.run(["readelf", "-d", target], capture_output=True, text=True, check=True).stdout
    assert "libtorch_cpu" in needed and "hip" not in needed
    script = """if True:
        import importlib.util, sys, torch
        spec = importlib.util.spec_from_file_location("_tpi_torch", sys.argv[1])
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        from terraform_provider_iterative_amd import ops
        from terraform_provider_iterative_amd.ops import _loader
        _loader._torch_ext = module
        out = ops.dropout(torch.ones(100, requires_grad=True), 0.5, ops.MaskStream(3))
        out.sum().backward()
        try:
            module.stream_and_capture(0)
        except ops.HipError as error:
            print(int(out.sum()), error)
    """
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, "-c", script, target], capture_output=True, text=True,
                         env=dict(os.environ, PYTHONPATH=root), timeout=120)
    want = int(ops.dropout(torch.ones(100), 0.5, (3, 0)).sum())
    assert res.stdout.startswith("%d this torch is not built for ROCm" % want), res.stdout + res.stderr


@pytest.mark.parametrize("shape", [(3 * (1 << 15) + 5,), (7, 41, 1031)])
@pytest.mark.parametrize("turned", [False, True])
def test_host_dropout_on_several_threads(shape, turned):
    """Ranges are split where they fall, inside a block of the generator and inside a row."""
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1))
    x = x.t() if turned and x.dim() == 2 else x.transpose(0, -1) if turned else x
    r = torch.randn(x.shape, generator=torch.Generator().manual_seed(2)).half().float()
    threads = torch.get_num_threads()
    try:
        results = []
        for count in (1, 2, 3, 5):
            torch.set_num_threads(count)
            results.append(ops.dropout(x, 0.3, KEY, residual=r))
    finally:
        torch.set_num_threads(threads)
    assert all(torch.equal(out, results[0]) for out in results)
    kept = torch.tensor(keep_mask(range(x.numel()), 0.3, *KEY)).reshape(x.shape)
    product = torch.where(kept, x.double() * (2 ** 32 / int(round(0.7 * 2 ** 32))), 0.0)
    # in 32 bits: the scale, the product and the sum are each rounded by half a step
    bound = 3 * 2.0 ** -24 * (product.abs() + r.double().abs())
    assert ((results[-1].double() - product - r.double()).abs() <= bound).all()


def test_the_host_operators_are_built_for_torchs_threads():
    """at::parallel_for compiled without OpenMP runs on one; the runtime is torch's, not a second."""
    import subprocess

    from terraform_provider_iterative_amd import _build

    if not torch.__config__.parallel_info().count("ATen parallel backend: OpenMP"):
        pytest.skip("torch itself does not use OpenMP")
    _build.build_torch_ext()
    names = subprocess.run(["nm", "-D", "--undefined-only", _build.TORCH_EXT], capture_output=True,
                           text=True, check=True).stdout
    needed = subprocess.run(["readelf", "-d", _build.TORCH_EXT], capture_output=True, text=True,
                            check=True).stdout
    assert "GOMP_parallel" in names and "omp" not in needed


# -- pools ---------------------------------------------------------------------------------------

def _pool():
    kv = torch.arange(2.0 * 10 * 4).reshape(2, 10, 4)
    pool = ops.PagePool(list(kv.unbind(0)), 4, 3, 5)
    pool.extend([0, 2], [9, 3])
    return pool


@pytest.mark.parametrize("how", ["deepcopy", "pickle", "state_dict"])
def test_a_copied_pool_has_books_and_pages_of_its_own(how):
    import copy
    import pickle

    pool = _pool()
    books, data = pool.meta.clone(), [t.clone() for t in pool.tensors]
    if how == "pickle":
        other = pickle.loads(pickle.dumps(pool))
    elif how == "deepcopy":
        other = copy.deepcopy(pool)
    else:  # as an attribute of a module that is copied
        module = torch.nn.Linear(2, 2)
        module.cache = pool
        other = copy.deepcopy(module).cache
    assert torch.equal(other.meta, books) and other.width == 5
    assert all(torch.equal(a, b) for a, b in zip(other.tensors, data))
    other.fork([0], [1])
    other.copy([0], [9])
    other.free([2])
    assert torch.equal(pool.meta, books) and all(torch.equal(a, b) for a, b in zip(pool.tensors, data))
    want = _pool()
    want.fork([0], [1])
    want.copy([0], [9])
    want.free([2])
    assert torch.equal(other.meta, want.meta)
    assert all(torch.equal(a, b) for a, b in zip(other.tensors, want.tensors))
    del pool
    other.compact(clear=True)
    want.compact(clear=True)
    assert torch.equal(other.meta, want.meta)


def test_a_shallow_copy_is_the_same_pool():
    import copy

    pool = _pool()
    other = copy.copy(pool)
    other.free([0])
    assert other.meta is pool.meta and pool.status()["live"] == 1


def test_bind_refuses_a_partial_page_of_two_sequences():
    """Either would go on writing in it; full pages may be shared, and a partial one of one sequence."""
    pool = ops.PagePool([torch.zeros(10, 4)], 4, 3, 5)
    before = pool.meta.clone()
    for table, lengths in (([[1, 2], [1, 2], [0, 0]], [7, 7, 0]),   # partial in both
                           ([[1, 2], [2, 3], [0, 0]], [7, 8, 0]),   # partial in one, full in the other
                           ([[1, 1], [2, 3], [0, 0]], [5, 8, 0])):  # both in one sequence
        with pytest.raises(ValueError, match="partial"):
            pool.bind(table, lengths)
        assert torch.equal(pool.meta, before)
    pool.bind([[1, 2], [1, 3], [1, 4]], [7, 5, 8])
    assert pool.refs.tolist() == [0, 3, 1, 1, 1] + [0] * 5
    pool.bind([[1, 2], [1, 2], [1, 2]], [8, 8, 4])
    assert pool.refs.tolist() == [0, 3, 2] + [0] * 7


def test_two_threads_compute_one_block_again_at_once():
    """Each backward pass over a graph is given the block's draws from the first on."""
    import threading

    masks = ops.MaskStream(3)
    first, again = masks.checkpoint_contexts()
    with first:
        drawn = [masks.next() for _ in range(4)]
    barrier, got = threading.Barrier(2, timeout=60), [[], []]

    def compute(out):
        with again:
            for _ in drawn:
                barrier.wait()
                out.append(masks.next())

    threads = [threading.Thread(target=compute, args=(out,)) for out in got]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert got[0] == got[1] == drawn and masks.number == 4


def test_draws_between_runs_of_a_recorded_step_follow_the_state():
    """The recorded program advances the state without the stream's knowing."""
    from torch.fx.experimental.proxy_tensor import make_fx

    masks, x = ops.MaskStream(3, device="cpu"), torch.ones(300)

    def step(v):
        out = ops.dropout(v, 0.5, masks)
        masks.advance()
        return out

    recorded = make_fx(step)(x)
    for _ in range(3):
        for _ in range(2):
            number = masks.state_dict()["number"]
            assert torch.equal(ops.dropout(x, 0.5, masks), ops.dropout(x, 0.5, (3, number)))
        masks.advance()
        number = masks.state_dict()["number"]
        assert torch.equal(recorded(x), ops.dropout(x, 0.5, (3, number)))
        assert masks.state_dict()["number"] == number + 1
        number = masks.state_dict()["number"]
        assert torch.equal(ops.dropout(x, 0.5, masks), ops.dropout(x, 0.5, (3, number)))
        recorded(x)
        number = masks.state_dict()["number"]
        assert torch.equal(ops.dropout(x, 0.5, masks), ops.dropout(x, 0.5, (3, number)))
        masks.advance()
