"""Operators on a rank's state on the MI355X (tests/test_device_state_ops.py) where they meet what
surrounds them: checkpoints, streams, transformations of a program."""
import pytest
import torch

from terraform_provider_iterative_amd import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _require_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")
    ops.hip(required=True)


def test_a_refusal_nobody_asked_for_is_still_there_after_a_resume():
    """What a resume does with books that hold a refusal: it goes on, and the next check raises."""
    pool = ops.PagePool([torch.zeros(8, 4, device="cuda")], 4, 3, 8)
    pool.extend(torch.tensor([0], device="cuda"), 100)
    saved = pool.meta.clone()
    again = ops.PagePool([torch.zeros(8, 4, device="cuda")], 4, 3, 8)
    again.meta.copy_(saved)
    again.resumed()
    with pytest.raises(ops.PageError, match="longer than a row"):
        again.check()
    again.extend(torch.tensor([0], device="cuda"), 10)
    again.check()
    other = ops.PagePool([torch.zeros(8, 4, device="cuda")], 2, 3, 8)
    other.meta.copy_(saved)
    with pytest.raises(ops.PageError, match="4 tokens a page"):
        other.resumed()


@pytest.mark.parametrize("as_tensor", [False, True])
def test_clearing_reaches_free_pages_that_a_copy_wrote(as_tensor):
    host, dev = [ops.PagePool([torch.ones(70, 9000, device=d)], 4, 2, 12) for d in ("cpu", "cuda")]
    for pool in (host, dev):
        pool.extend([0], 10)
        pool.compact(clear=True)
        for src, dst in (([0, 1], [69, 2]), ([69], [33])):
            if as_tensor and pool is dev:
                src, dst = (torch.tensor(v, device="cuda") for v in (src, dst))
            pool.copy(src, dst)
        assert pool.tensors[0][[33, 69]].all()
    assert torch.equal(host.meta[8:], dev.meta[8:].cpu())
    for pool in (host, dev):
        pool.compact(clear=True)
        assert pool.tensors[0][:3].all() and not pool.tensors[0][3:].any()
    assert torch.equal(host.meta[8:], dev.meta[8:].cpu())


@pytest.mark.parametrize("act", ["extend", "fork"])
def test_of_two_reasons_the_same_is_given_every_time(act):
    """More entries than the small plan takes, a slot named twice and too few pages: as on every run,
    and as for few entries, the reason with the higher number."""
    pool = ops.PagePool([torch.zeros(700, 4, device="cuda")], 4, 3000, 700)
    if act == "fork":
        pool.extend([0], 3)  # a partial page: each fork takes one
    slots = torch.arange(1, 1501, device="cuda")
    slots[1499] = 5
    source = torch.zeros_like(slots)
    for _ in range(20):
        if act == "extend":
            pool.extend(slots, 1)
        else:
            pool.fork(source, slots)
        assert pool.status()["error"] == "a slot is named twice"
        with pytest.raises(ops.PageError, match="named twice"):
            pool.check()
    slots[1499] = 1500
    pool.extend(slots, 1) if act == "extend" else pool.fork(source, slots)
    with pytest.raises(ops.PageError, match="not enough free pages"):
        pool.check()
    assert pool.status()["live"] == (act == "fork")


# -- transformations of a program ------------------------------------------------------------------

@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
def test_a_graph_of_dropout_computes_dropout(mode):
    from torch.fx.experimental.proxy_tensor import make_fx

    def block(x):
        x = x.detach().requires_grad_(True)
        out = ops.dropout(x * 2, 0.4, (3, 7), residual=x.float())
        return out.detach(), torch.autograd.grad(out.sum(), x)[0]

    make = lambda d: torch.randn(6, 11, generator=torch.Generator().manual_seed(1)).bfloat16().to(d)
    traced = make_fx(block, tracing_mode=mode)(torch.zeros(6, 11, dtype=torch.bfloat16, device="cuda"))
    for got, want, host in zip(traced(make("cuda")), block(make("cuda")), block(make("cpu"))):
        assert torch.equal(got, want) and torch.equal(got.cpu(), host)


def test_dropout_refuses_tensors_without_memory():
    """Refused on the host, before anything is launched."""
    x = torch.ones(8, 4, device="cuda")
    freed = torch.ones(8, 4, device="cuda")
    freed.untyped_storage().resize_(0)
    for call in (lambda: ops.dropout(freed, 0.5, (1, 2)),
                 lambda: ops.dropout(x, 0.5, (1, 2), residual=freed),
                 lambda: ops.PagePool([x, freed], 4, 2)):
        with pytest.raises(ValueError, match="memory of their own"):
            call()


@pytest.mark.parametrize("residual", [False, True])
def test_forward_mode_carries_the_tangents(residual):
    import torch.autograd.forward_ad as forward

    x, tx, r, tr = (torch.randn(65, 33, generator=torch.Generator().manual_seed(i)).bfloat16()
                    for i in range(4))
    masks = ops.MaskStream(4, device="cuda")
    with forward.dual_level():
        out = ops.dropout(forward.make_dual(x.cuda(), tx.cuda()), 0.4, masks,
                          residual=forward.make_dual(r.cuda(), tr.cuda()) if residual else None)
        primal, tangent = forward.unpack_dual(out)
    assert torch.equal(primal.cpu(), ops.dropout(x, 0.4, (4, 0), residual=r if residual else None))
    assert torch.equal(tangent.cpu(), ops.dropout(tx, 0.4, (4, 0), residual=tr if residual else None))


# -- blocks that are computed twice ----------------------------------------------------------------

@pytest.mark.parametrize("captured", [False, True])
def test_a_block_computed_twice_after_the_stream_has_advanced(captured):
    """Activation checkpointing with the draw taken outside; in a graph every replay draws anew."""
    from torch.utils.checkpoint import checkpoint

    masks = ops.MaskStream(21, device="cuda")
    w = torch.randn(64, 64, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_(True)
    x = torch.randn(32, 64, generator=torch.Generator().manual_seed(2)).cuda().requires_grad_(True)

    def block(v, draw):
        return (ops.dropout(v * w[0], 0.5, draw) * w[1]).pow(2)

    def step(one, two):
        y = checkpoint(block, checkpoint(block, x, one, use_reentrant=False), two, use_reentrant=False)
        if one is not None and isinstance(one, ops.Draw) and one.state is not None:
            masks.advance()
        return torch.autograd.grad(y.sum(), (x, w))

    def check(got, number):
        want = step((21, number), (21, number + 1))
        assert all(torch.equal(g, v) for g, v in zip(got, want))

    if not captured:
        for number in range(0, 6, 2):
            check(step(masks.next(), masks.next()), number)
        return
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(masks.next(), masks.next())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(masks.next(), masks.next())
    for replay in range(4):
        graph.replay()
        torch.cuda.synchronize()
        check(got, 2 + 2 * replay)
        assert masks.state_dict()["number"] == 4 + 2 * replay


def test_draws_of_a_step_in_several_graphs_and_streams():
    """A step whose draws are captured in two graphs, with eager ones of the same step before and
    between: none of them refers to what another capture, or an eager draw, has copied."""
    masks, x = ops.MaskStream(5, device="cuda"), torch.ones(512, device="cuda")
    ops.dropout(x, 0.5, masks)  # draw 0 of the step, eager
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        a = ops.dropout(x, 0.5, masks)
    with torch.cuda.graph(two):
        b = ops.dropout(x, 0.5, masks)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = ops.dropout(x, 0.5, masks)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(c, ops.dropout(x, 0.5, (5, 3)))
    for step in range(3):
        for order in ((one, two), (two, one)):
            for graph in order:
                graph.replay()
            assert torch.equal(a, ops.dropout(x, 0.5, (5, 4 * step + 1)))
            assert torch.equal(b, ops.dropout(x, 0.5, (5, 4 * step + 2)))
        if step == 0:
            masks.advance()
        else:
            masks.state[1:].add_(4)  # as a step of four draws would


@pytest.mark.parametrize("device", [None, "cuda"])
@pytest.mark.parametrize("captured", [False, True])
def test_checkpointed_layers_draw_the_same_masks_twice(device, captured):
    from torch.utils.checkpoint import checkpoint

    if captured and device is None:
        pytest.skip("a stream without a device is refused in a capture")
    masks = ops.MaskStream(9, device=device)
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(64, 64), ops.CounterDropout(0.5, masks),
                                torch.nn.Linear(64, 64), ops.CounterDropout(0.3, masks)).cuda()
    x = torch.randn(32, 64, generator=torch.Generator().manual_seed(2)).cuda().requires_grad_(True)
    inputs = [x, *model.parameters()]

    def step():
        y = checkpoint(model, x, use_reentrant=False, context_fn=masks.checkpoint_contexts)
        if device:
            masks.advance()
        return torch.autograd.grad(y.pow(2).sum(), inputs)

    def check(got, number):
        a = ops.dropout(model[0](x), 0.5, (9, number))
        b = ops.dropout(model[2](a), 0.3, (9, number + 1))
        want = torch.autograd.grad(b.pow(2).sum(), inputs)
        assert all(torch.equal(g, w) for g, w in zip(got, want))
        assert masks.state_dict()["number"] == number + 2

    if not captured:
        for number in (0, 2, 4):
            check(step(), number)
        return
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for replay in range(4):
        graph.replay()
        torch.cuda.synchronize()
        check(got, 2 + 2 * replay)


def test_a_second_computation_without_the_contexts_is_refused():
    from torch.utils.checkpoint import checkpoint

    masks = ops.MaskStream(3, device="cuda")
    x = torch.randn(64, device="cuda", requires_grad=True)
    y = checkpoint(lambda v: ops.dropout(v, 0.5, masks).pow(2), x, use_reentrant=False)
    with pytest.raises(RuntimeError, match="computes again"):
        y.sum().backward()
    assert masks.state_dict()["number"] == 1


# -- errors, streams, memory -----------------------------------------------------------------------

def test_an_earlier_calls_error_is_not_a_launchs():
    """What another caller has left in the runtime's last error neither fails an operation nor leaves
    out a part of it."""
    import ctypes

    from terraform_provider_iterative_amd import _build

    runtime = ctypes.CDLL(_build.HIP_SO)  # finds the runtime that the library is linked to
    x = torch.ones(1000, device="cuda")
    pool = ops.PagePool([torch.ones(32, 64, device="cuda")], 4, 8, 8)
    slots = [torch.tensor(v, device="cuda") for v in ([0], [1, 2], [0, 0])]
    torch.cuda.synchronize()
    calls = [lambda: ops.dropout(x, 0.5, (1, 2)), lambda: pool.extend(slots[0], 7),
             lambda: pool.fork(slots[2], slots[1]), lambda: pool.free(slots[0]),
             lambda: pool.copy(slots[0], slots[1][:1]), lambda: pool.compact(clear=True)]
    for call in calls:
        assert runtime.hipSetDevice(1 << 20) != 0  # refused, and remembered
        try:
            call()
        finally:
            assert runtime.hipGetLastError() != 0  # still there for whoever asks
    assert pool.status() == {"pages": 32, "free": 29, "live": 3, "error": None}
    assert pool.lengths.tolist() == [0, 7, 7] + [0] * 5


@pytest.mark.parametrize("captured", [False, True])
def test_a_dropped_pools_memory_waits_for_a_side_stream(captured):
    """Nothing that a pool allocated, nor its tensors, is given to another tensor while work that the
    pool has enqueued on a side stream may still use it."""
    side = torch.cuda.Stream()
    pool = ops.PagePool([torch.ones(5000, 1 << 12, device="cuda")], 4, 16, 5000)
    pool.extend([0, 1], [8000, 8000])
    pool.free([0])
    held = {t.data_ptr(): t.numel() for t in (pool.meta, pool._scratch, pool._chunk, pool.tensors[0])}
    torch.cuda.synchronize()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            pool.compact()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # some tenths of a second
        pool.compact(clear=True)
    del pool
    other = [torch.empty(n, dtype=torch.int32 if n < 1 << 24 else torch.float32, device="cuda")
             for n in held.values()]
    assert not side.query()
    assert not set(held) & {t.data_ptr() for t in other}
    torch.cuda.synchronize()


def test_a_refused_call_leaves_no_error_behind():
    """What the library has reported is not found again by the next one who asks the runtime."""
    import ctypes

    from terraform_provider_iterative_amd import _build

    runtime = ctypes.CDLL(_build.HIP_SO)
    torch.cuda.synchronize()
    assert runtime.hipGetLastError() == 0
    lib = ops.hip()
    with pytest.raises(ops.HipError, match="hipHostRegister"):  # of no memory
        lib.check(lib.tpi_host_register(None, 0), "hipHostRegister")
    assert runtime.hipGetLastError() == 0
    assert torch.zeros(3, device="cuda").tolist() == [0.0] * 3


def test_draws_between_replays_follow_the_state():
    """A replay advances the state without the stream's knowing: an eager draw after it, also of a step
    that has drawn before it, has the number that state_dict() names."""
    masks, x = ops.MaskStream(5, device="cuda"), torch.ones(512, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = ops.dropout(x, 0.5, masks)
        masks.advance()
    for _ in range(3):
        for _ in range(2):
            number = masks.state_dict()["number"]
            assert torch.equal(ops.dropout(x, 0.5, masks), ops.dropout(x, 0.5, (5, number)))
            start = int(masks.state[1])
            graph.replay()
            assert torch.equal(a, ops.dropout(x, 0.5, (5, start)))
        masks.advance()
