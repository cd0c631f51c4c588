"""Dropout from a counter-based generator and the pages of a paged cache, on the host.

The oracles are written from the definitions: Philox in Python integers, a pool as dictionaries.
"""
import numpy as np
import pytest
import torch

from state_oracles import PoolOracle, dropout_oracle, keep_mask, philox4x32
from terraform_provider_iterative_amd import ops
from terraform_provider_iterative_amd.checkpoint import TrainingState
from terraform_provider_iterative_amd.ops import masking, paging

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def rounding(value, dtype):
    """The most that one rounding of ``value`` to ``dtype`` can change it: half a step, relative
    in the normal range, and the smallest normal number's half step below it (there steps do not
    shrink any more: fp16 values under 2^-14 are all multiples of 2^-24)."""
    f = torch.finfo(dtype)
    return value.abs().clamp(min=f.tiny) * f.eps / 2


# -- the generator -------------------------------------------------------------------------------

def test_philox_known_answers():
    """The published generator's known answers for 10 rounds (all zeros, all ones, digits of pi)."""
    ones = 0xFFFFFFFF
    assert philox4x32((0, 0, 0, 0), (0, 0)) == (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)
    assert philox4x32((ones,) * 4, (ones,) * 2) == (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)
    assert philox4x32((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) \
        == (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)


def test_argument_blocks_match_the_c_structs():
    assert paging._POOL.size == ops.native().PAGES_SIZE
    assert paging._CHUNK.itemsize == ops.native().PAGE_CHUNK_SIZE


@pytest.mark.parametrize("p", [0.0, 1e-9, 0.1, 0.5, 0.75, 1 - 2 ** -20, 1.0])
def test_kept_elements_are_the_definitions(p):
    n = 20001
    got = ops.dropout(torch.ones(n), p, (0x0123456789ABCDEF, 0x123456789)) != 0
    assert got.tolist() == keep_mask(range(n), p, 0x0123456789ABCDEF, 0x123456789)


def test_the_low_half_decides_ties():
    """Where the first half-word equals the threshold's high half, the second one decides: such
    elements are found among many, and both outcomes occur."""
    n, p, key = 1 << 21, 0.3, (5, 9)
    kept = ops.dropout(torch.ones(n), p, key) != 0
    threshold, _ = masking.keep_threshold(p)
    fine = ops.dropout(torch.ones(n), 1 - (threshold >> 16) / 65536, key) != 0  # low half 0
    extra = (kept & ~fine).nonzero().flatten().tolist()
    coarse = ops.dropout(torch.ones(n), 1 - ((threshold >> 16) + 1) / 65536, key) != 0
    ties = (coarse & ~fine).nonzero().flatten().tolist()
    assert len(ties) > 10 and 0 < len(extra) < len(ties)
    assert [bool(v) for v in kept[ties]] == keep_mask(ties, p, *key)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [None, "same", torch.float32])
def test_dropout_forward_and_gradients(dtype, residual):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 37, 19, generator=g).to(dtype).requires_grad_(True)
    r = None
    if residual is not None:
        kind = dtype if residual == "same" else residual
        r = torch.randn(3, 37, 19, generator=g).to(kind).requires_grad_(True)
    out = ops.dropout(x, 0.3, (11, 2), residual=r)
    grad = torch.randn(out.shape, generator=g).to(out.dtype)
    kept, want = dropout_oracle(x, 0.3, (11, 2), r)
    # one rounding of the product and of the sum in 32 bits, one to the output's type: each at most
    # half a step of a value no larger than |product| + |residual|
    size = (want - (0 if r is None else r.detach().double())).abs() + \
        (0 if r is None else r.detach().double().abs())
    bound = size * 3 * 2.0 ** -24 + rounding(size, out.dtype)
    assert out.dtype == (dtype if r is None else r.dtype)
    assert ((out.detach().double() - want).abs() <= bound).all()
    assert ((out != 0) == kept).all() if r is None else True
    inputs = (x,) if r is None else (x, r)
    grads = torch.autograd.grad(out, inputs, grad)
    scale = float(masking.keep_threshold(0.3)[1])
    dx = torch.where(kept, grad.double() * scale, 0.0)
    assert grads[0].dtype == dtype
    assert ((grads[0].double() - dx).abs() <= dx.abs() * 2 * 2.0 ** -24 + rounding(dx, dtype)).all()
    if r is not None:
        assert torch.equal(grads[1], grad)


def test_dropout_gradient_against_differences():
    x = torch.randn(64, generator=torch.Generator().manual_seed(0)).requires_grad_(True)
    w = torch.randn(64, generator=torch.Generator().manual_seed(1))

    def loss(v):
        return (ops.dropout(v, 0.4, (3, 4)).double() * w.double()).sum()

    grad, = torch.autograd.grad(loss(x), x)
    step = 0.5  # the operator is linear: any step does, a large one loses least to rounding
    for i in range(64):
        e = torch.zeros(64)
        e[i] = step
        diff = (loss(x.detach() + e) - loss(x.detach() - e)) / (2 * step)
        assert abs(float(diff) - float(grad[i])) < 1e-5


def test_dropout_can_be_differentiated_twice():
    x = torch.randn(50, requires_grad=True)
    y = ops.dropout(x, 0.5, (1, 1))
    g, = torch.autograd.grad((y ** 2).sum(), x, create_graph=True)
    gg, = torch.autograd.grad(g.sum(), x)
    kept, _ = dropout_oracle(x, 0.5, (1, 1))
    assert torch.allclose(gg, torch.where(kept, 8.0, 0.0))  # 2 scale^2


def test_dropped_elements_are_zero_whatever_they_hold():
    n = 4096
    kept = torch.tensor(keep_mask(range(n), 0.5, 7, 0))
    for bad in (float("nan"), float("inf"), -float("inf")):
        x = torch.where(kept, 1.0, bad)
        out = ops.dropout(x, 0.5, (7, 0))
        assert torch.equal(out, torch.where(kept, 2.0, 0.0))
    out = ops.dropout(torch.full((n,), float("nan")), 0.5, (7, 0))
    assert torch.equal(out.isnan(), kept)


@pytest.mark.parametrize("view", ["t", "slice", "expand", "permute", "step", "rows"])
def test_views_are_masked_by_their_logical_index(view):
    base = torch.randn(12, 10, 14, generator=torch.Generator().manual_seed(3))
    x = {"t": base[0].t(), "slice": base[:, 2:7, 1:], "permute": base.permute(2, 0, 1),
         "expand": base[:, :1].expand(12, 5, 14), "step": base[::2, :, ::3],
         "rows": base[:, :, 3:11]}[view]
    want = ops.dropout(x.contiguous(), 0.4, (2, 3))
    assert torch.equal(ops.dropout(x, 0.4, (2, 3)), want)
    r = torch.randn(x.shape, generator=torch.Generator().manual_seed(4))
    want = ops.dropout(x.contiguous(), 0.4, (2, 3), residual=r)
    assert torch.equal(ops.dropout(x, 0.4, (2, 3), residual=r), want)
    turned = r.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ops.dropout(x, 0.4, (2, 3), residual=turned), want)


def test_lazily_negated_views():
    z = torch.view_as_complex(torch.randn(100, 2, generator=torch.Generator().manual_seed(3)))
    x = torch.conj(z).imag
    assert x.is_neg()
    want = ops.dropout(-z.imag.contiguous(), 0.3, (1, 2))
    assert torch.equal(ops.dropout(x, 0.3, (1, 2)), want)
    assert torch.equal(ops.dropout(torch.zeros(100), 0.3, (1, 2), residual=x), -z.imag)


def test_the_gradient_of_an_expanded_residual_is_summed():
    x, r = torch.randn(5, 7, requires_grad=True), torch.randn(7, requires_grad=True)
    out = ops.dropout(x, 0.3, (1, 2), residual=r.expand(5, 7))
    grad = torch.randint(-8, 9, (5, 7)).float()
    dx, dr = torch.autograd.grad(out, (x, r), grad)
    assert torch.equal(dr, grad.sum(0)) and torch.equal(dx, ops.dropout(grad, 0.3, (1, 2)))
    same, = torch.autograd.grad(ops.dropout(x, 0.3, (1, 2), residual=x), x, grad)
    assert torch.equal(same, dx + grad)


@pytest.mark.parametrize("starts,shape", [((0, 0, 0), (4, 6, 33)), ((1, 2, 5), (2, 3, 17)),
                                          ((3, 5, 32), (1, 1, 1)), ((0, 0, 16), (4, 6, 8))])
def test_a_shard_has_the_wholes_mask(starts, shape):
    whole = torch.randn(4, 6, 33, generator=torch.Generator().manual_seed(3))
    want = ops.dropout(whole, 0.4, (2, 3))
    part = tuple(slice(a, a + n) for a, n in zip(starts, shape))
    x = whole[part].contiguous().requires_grad_(True)
    got = ops.dropout(x, 0.4, (2, 3), shard=((4, 6, 33), starts))
    assert torch.equal(got, want[part])
    grad, = torch.autograd.grad(got, x, torch.ones(shape))
    assert torch.equal(grad != 0, got != 0)


def test_indexes_beyond_32_bits():
    whole, starts = (1 << 20, 1 << 20), ((1 << 20) - 2, (1 << 20) - 100)
    got = ops.dropout(torch.ones(2, 100), 0.5, (1, 2), shard=(whole, starts)) != 0
    index = [(starts[0] + r) * whole[1] + starts[1] + c for r in range(2) for c in range(100)]
    assert index[0] > 1 << 39
    assert got.flatten().tolist() == keep_mask(index, 0.5, 1, 2)


@pytest.mark.parametrize("shape", [(0,), (3, 0), (), (1,), (7,)])
def test_dropout_of_few_elements(shape):
    x = torch.randn(shape).requires_grad_(True)
    out = ops.dropout(x, 0.5, (1, 2))
    assert out.shape == x.shape
    grad, = torch.autograd.grad(out.sum(), x)
    kept = torch.tensor(keep_mask(range(x.numel()), 0.5, 1, 2), dtype=torch.bool).reshape(shape)
    assert torch.equal(grad, torch.where(kept, 2.0, 0.0))


def test_dropout_refusals():
    x = torch.ones(4, 4)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            ops.dropout(x, p, (0, 0))
    with pytest.raises(TypeError):
        ops.dropout(x.double(), 0.1, (0, 0))
    with pytest.raises(TypeError):
        ops.dropout([1.0], 0.1, (0, 0))
    with pytest.raises(TypeError):
        ops.dropout(x, 0.1, 3)
    for draw in ((-1, 0), (1 << 64, 0), (0, -1), (0, 1 << 63)):
        with pytest.raises(ValueError):
            ops.dropout(x, 0.1, draw)
    with pytest.raises(ValueError):
        ops.dropout(x, 0.1, (0, 0), residual=torch.ones(4))
    with pytest.raises(TypeError):
        ops.dropout(x, 0.1, (0, 0), residual=x.half())
    for shard in (((4,), (0,)), ((4, 4), (1, 0)), ((8, 8), (-1, 0)), ((1 << 40, 1 << 40), (0, 0))):
        with pytest.raises(ValueError):
            ops.dropout(x, 0.1, (0, 0), shard=shard)
    with pytest.raises(ValueError):  # no two of 7 dimensions can be walked as one
        big = torch.zeros([3] * 7)[tuple([slice(0, 2)] * 7)]
        ops.dropout(big, 0.1, (0, 0))
    with pytest.raises(ValueError):
        ops.dropout(x, 0.1, ops.Draw(0, 0, torch.zeros(1, dtype=torch.int64)))


# -- streams of masks ------------------------------------------------------------------------------

@pytest.mark.parametrize("device", [None, "cpu"])
def test_a_stream_numbers_its_draws_and_resumes(device):
    x = torch.ones(1000)
    a = ops.MaskStream(9, device=device)
    first = [ops.dropout(x, 0.5, a) for _ in range(3)]
    assert not torch.equal(first[0], first[1])
    assert [torch.equal(v, ops.dropout(x, 0.5, (9, i))) for i, v in enumerate(first)] == [True] * 3
    saved = a.state_dict()
    assert saved == {"seed": 9, "number": 3}
    later = [ops.dropout(x, 0.5, a) for _ in range(2)]
    b = ops.MaskStream(1, device=device)
    b.load_state_dict(saved)
    assert all(torch.equal(v, ops.dropout(x, 0.5, b)) for v in later)


def test_a_device_streams_backward_keeps_its_draw():
    masks = ops.MaskStream((1 << 64) - 3, device="cpu")
    x = torch.randn(500, requires_grad=True)
    y = ops.dropout(x, 0.5, masks)
    z = ops.dropout(x, 0.5, masks)
    masks.advance()  # the next step has begun when this one's backward pass runs
    for number, out in enumerate((y, z)):
        grad, = torch.autograd.grad(out.sum(), x)
        assert torch.equal(grad, ops.dropout(torch.ones(500), 0.5, ((1 << 64) - 3, number)))
    assert masks.state_dict() == {"seed": (1 << 64) - 3, "number": 2}
    assert torch.equal(ops.dropout(x, 0.5, masks).detach(),
                       ops.dropout(x.detach(), 0.5, ((1 << 64) - 3, 2)))
    with pytest.raises(ValueError):
        ops.MaskStream(0).advance()


def test_the_layer_and_evaluation():
    masks = ops.MaskStream(4)
    layer = ops.CounterDropout(0.25, masks)
    x, r = torch.randn(8, 8), torch.randn(8, 8)
    assert torch.equal(layer(x, r), ops.dropout(x, 0.25, (4, 0), residual=r))
    layer.eval()
    assert layer(x) is x and torch.equal(layer(x, r), x + r)
    assert masks.number == 1
    with pytest.raises(ValueError):
        ops.CounterDropout(2.0, masks)


# -- pages -------------------------------------------------------------------------------------------

def _tensors(kind, pages, g):
    """Pools of several layouts, with the page index of each byte in it."""
    if kind == "kv":
        return list(torch.randn(4, pages, 4, 2, 8, generator=g).unbind(0))
    if kind == "odd":
        return [torch.randint(0, 255, (pages, 13, 3), dtype=torch.uint8, generator=g),
                torch.randn(pages, 7, generator=g).half()]
    if kind == "heads":  # [heads, pages, ...] storage
        return [torch.randn(3, pages, 4, 5, generator=g).transpose(0, 1)]
    return [torch.randn(pages, 2, 4, 8, generator=g).to(torch.bfloat16)[:, i] for i in range(2)]


def _agree(pool, oracle):
    assert pool.table.tolist() == oracle.table.tolist()
    assert pool.lengths.tolist() == oracle.lengths.tolist()
    assert pool.refs.tolist() == oracle.refs.tolist()
    assert pool.status() == {"pages": pool.pages, "free": oracle.free_count(),
                             "live": pool.pages - oracle.free_count(), "error": None}
    for got, want in zip(pool.tensors, oracle.tensors):
        assert torch.equal(got, want)


@pytest.mark.parametrize("kind", ["kv", "odd", "heads", "interleaved"])
@pytest.mark.parametrize("tokens,pages,slots,width", [(4, 40, 9, 12), (1, 70, 5, 70), (16, 33, 40, 3)])
def test_operations_agree_with_the_oracle(kind, tokens, pages, slots, width):
    g = torch.Generator().manual_seed(pages)
    rng = np.random.RandomState(slots)
    tensors = _tensors(kind, pages, g)
    oracle = PoolOracle([t.clone() for t in tensors], tokens, slots, width)
    pool = ops.PagePool(tensors, tokens, slots, width)
    _agree(pool, oracle)
    done = {}
    for _ in range(120):
        act, args = oracle.random_call(rng)
        error = oracle.refusal(act, *args)
        if error:
            before = pool.meta.clone()
            with pytest.raises(ops.PageError, match=error):
                getattr(pool, act)(*args)
            assert torch.equal(pool.meta, before)
        else:
            getattr(pool, act)(*args)
            getattr(oracle, act)(*args)
        done[act, error or ""] = done.get((act, error or ""), 0) + 1
        _agree(pool, oracle)
    assert {"extend", "fork", "free", "compact"} <= {a for (a, e) in done if not e}


def test_lists_are_checked_at_once():
    pool = ops.PagePool([torch.zeros(8, 4)], 4, 3, 4)
    for call in (lambda: pool.extend([3], 1), lambda: pool.extend([-1], 1),
                 lambda: pool.extend([0, 0], 1), lambda: pool.extend([0], [1, 2]),
                 lambda: pool.extend([0], -1), lambda: pool.extend([0], [-1]),
                 lambda: pool.extend([0, 1, 2, 0], 1), lambda: pool.fork([0], [1, 2]),
                 lambda: pool.fork([0, 0], [1, 1]), lambda: pool.free([7]),
                 lambda: pool.copy([0], [8]), lambda: pool.copy([0, 1], [2, 2]),
                 lambda: pool.copy([0, 1], [1, 2]), lambda: pool.copy([0], [])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        pool.free(torch.tensor([0.0]))
    with pytest.raises(TypeError):
        pool.free(torch.tensor([[0]]))
    assert pool.status()["free"] == 8
    pool.copy([], [])
    pool.free([])
    pool.extend([], 5)
    pool.fork([], [])


def test_a_pool_refuses_what_it_cannot_hold():
    ok = torch.zeros(8, 4)
    for args in (([], 4, 3), ([ok, torch.zeros(9, 4)], 4, 3), ([torch.zeros(8)], 4, 3),
                 ([torch.zeros(8, 0)], 4, 3), ([ok], 0, 3), ([ok], 4, 0), ([ok], 4, 3, 0),
                 ([ok[:, :1].expand(8, 4)], 4, 3), ([torch.zeros(8, 3, 4, 5)[:, :2, :2, :2]], 4, 3),
                 ([torch.zeros(20).as_strided((8, 4), (2, 1))], 4, 3),
                 ([torch.zeros(8, 4, requires_grad=True)], 4, 3)):
        with pytest.raises(ValueError):
            ops.PagePool(*args)


def test_bind_takes_over_a_table():
    table = [[5, 2, -1], [-1, -1, -1], [5, 0, 7]]
    pool = ops.PagePool([torch.arange(32.0).reshape(8, 4)], 4, 3, 4)
    pool.bind(table, [6, 0, 12])
    assert pool.refs.tolist() == [1, 0, 1, 0, 0, 2, 0, 1]
    assert pool.table.tolist() == [[5, 2, -1, -1], [-1] * 4, [5, 0, 7, -1]]
    pool.compact(clear=True)
    assert pool.table.tolist() == [[1, 2, -1, -1], [-1] * 4, [1, 0, 3, -1]]
    assert pool.tensors[0][:4].tolist() == torch.arange(32.0).reshape(8, 4)[[0, 5, 2, 7]].tolist()
    assert not pool.tensors[0][4:].any()
    for bad in (([[8, 0, 0]] * 3, [1, 1, 1]), ([[0, 0, 0]] * 3, [13, 0, 0]),
                ([[0, 0, 0]] * 2, [0, 0]), ([[0] * 5] * 3, [0, 0, 0]), ([[0, 0, 0]] * 3, [-1, 0, 0]),
                ([[-1, 0, 0]] * 3, [1, 0, 0])):
        with pytest.raises(ValueError):
            pool.bind(*bad)


def test_books_of_another_pool_are_refused():
    pools = [ops.PagePool([torch.zeros(8, 4)], 4, slots, width) for slots, width in ((4, 8), (8, 4))]
    assert pools[0].meta.numel() != pools[1].meta.numel()
    other = ops.PagePool([torch.zeros(8, 4)], 8, 4, 8)
    other.extend([1], 9)
    pools[0].meta.copy_(other.meta)
    with pytest.raises(ops.PageError, match="8 tokens a page"):
        pools[0].check()


def test_clearing_leaves_pages_that_are_zero_already():
    """Only pages that were free and written, or that were freed, are cleared again."""
    data = torch.ones(16, 4)
    pool = ops.PagePool([data], 4, 2, 16)
    pool.extend([0], 10)
    pool.compact(clear=True)
    assert data[3:].sum() == 0 and data[:3].sum() == 12
    data[8] = 3.0  # written behind the pool's back: not the pool's business
    pool.extend([1], 4)
    data[3] = 5.0
    pool.free([0])
    pool.compact(clear=True)
    assert data[0].tolist() == [5.0] * 4 and pool.table[1, 0] == 0
    assert data[1:8].sum() == 0 and data[8:].sum() == 12


# -- checkpoints ---------------------------------------------------------------------------------

def test_a_checkpoint_carries_the_masks_and_the_pages(tmp_path):
    """A rank that trains with dropout and samples from a paged cache goes on bit for bit."""
    def build():
        torch.manual_seed(0)
        model = torch.nn.Linear(16, 16)
        opt = torch.optim.AdamW(model.parameters(), lr=1e-2)
        model(torch.zeros(1, 16)).sum().backward()
        opt.step()
        masks = ops.MaskStream(3)
        kv = torch.zeros(2, 12, 4, 8)
        pool = ops.PagePool(list(kv.unbind(0)), 4, 4, 6)
        state = TrainingState(model, opt, path=str(tmp_path / "spill"), tile_bytes=4096,
                              stateful={"masks": masks}, paged={"kv": pool})
        return model, opt, masks, kv, pool, state

    def step(model, opt, masks, kv, pool, i):
        if i % 3 == 0:
            pool.extend([i % 4], 5)
            page = int(pool.table[i % 4, (int(pool.lengths[i % 4]) - 1) // 4])
            kv[:, page] = float(i + 1)
        if i == 4:
            pool.fork([0], [2])
        if i == 5:
            pool.free([0])
        x = torch.randn(4, 16)
        opt.zero_grad()
        ops.dropout(model(x), 0.5, masks, residual=x).pow(2).mean().backward()
        opt.step()

    def sequences(kv, pool):
        return [[kv[:, page].clone() for page in row if page >= 0] for row in pool.table.tolist()]

    run = build()
    for i in range(6):
        step(*run[:5], i)
    run[5].save({"step": 6})
    pool, kv = run[4], run[3]
    live = pool.status()["live"]
    assert (pool.refs[:live] > 0).all() and not kv[:, live:].any()
    for i in range(6, 9):
        step(*run[:5], i)
    run[5].close()

    again = build()
    for t in (again[3], again[4].meta):
        t.fill_(7)  # whatever the successor's memory holds
    assert again[5].resume()["step"] == 6
    for i in range(6, 9):
        step(*again[:5], i)
    for a, b in zip(run[0].parameters(), again[0].parameters()):
        assert torch.equal(a, b)
    assert torch.equal(run[4].meta, again[4].meta)
    for a, b in zip(sequences(run[3], run[4]), sequences(again[3], again[4])):
        assert len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))
    again[5].close()


def test_the_training_example_draws_the_same_masks_after_a_resume(tmp_path):
    """examples/train with --dropout: stopped after 5 steps and resumed, its last step draws what
    an uninterrupted run's does and comes to the same loss."""
    import os
    import re
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

    def train(name, *steps):
        os.makedirs(tmp_path / name, exist_ok=True)
        for n in steps:
            res = subprocess.run(
                [sys.executable, os.path.join(root, "examples", "train", "train.py"), "--hidden",
                 "32", "--layers", "2", "--batch", "2", "--seq", "8", "--dropout", "0.2", "--steps",
                 str(n)], capture_output=True, text=True, timeout=300,
                env=dict(os.environ, TPI_DATA_DIRECTORY=str(tmp_path / name), OMP_NUM_THREADS="1"))
            assert res.returncode == 0, res.stdout + res.stderr
        return re.findall(r"step 8 loss (\S+)", res.stdout), (tmp_path / name / ".ckpt-rank0")

    from terraform_provider_iterative_amd.checkpoint.checkpointer import describe_checkpoint

    (a, whole), (b, resumed) = train("whole", 8), train("resumed", 5, 8)
    assert a and a == b
    states = [describe_checkpoint(str(path))["metadata"]["training_state"]["stateful"]["masks"]
              for path in (whole, resumed)]
    assert states[0] == states[1] and states[0]["number"] == 18  # 2 a step, and the warm step's


RANK_LOOP = r'''#!%(python)s
import hashlib, os, signal, sys
sys.path.insert(0, %(root)r)
import torch
from terraform_provider_iterative_amd import ops
from terraform_provider_iterative_amd.checkpoint import TrainingState

WHERE = os.environ.get("KILL_WHERE", "none")
first = os.environ.get("TPI_RESTART_COUNT", "0") == "0"
torch.set_num_threads(1)
torch.manual_seed(0)
masks = ops.MaskStream(5)
model = torch.nn.Sequential(torch.nn.Linear(16, 32), ops.CounterDropout(0.3, masks),
                            torch.nn.Linear(32, 16))
opt = torch.optim.AdamW(model.parameters(), lr=1e-2)
model(torch.zeros(1, 16)).sum().backward()
opt.step()
kv = torch.zeros(3, 40, 4, 16)
pool = ops.PagePool(list(kv.unbind(0)), page_tokens=4, slots=6, width=10)
state = TrainingState(model, opt, path=os.path.join(os.environ.get("TPI_DATA_DIRECTORY", "."),
                                                   ".spill"), tile_bytes=4096,
                      stateful={"masks": masks}, paged={"kv": pool})
state.resume()
start = state.step_value or 0
print("start", start, "live", pool.status()["live"], flush=True)
state.install()

def kill(where, step):
    if first and where == WHERE and step == 6:
        os.kill(os.getpid(), signal.SIGTERM)

def append(slots, rows):  # one token each
    pool.extend(slots, 1)
    for slot, row in zip(slots, rows):
        at = int(pool.lengths[slot]) - 1
        kv[:, int(pool.table[slot, at // 4]), at %% 4] = row

for step in range(start, 12):
    x = torch.randn(6, 16)
    y = ops.dropout(model(x), 0.2, masks, residual=x)
    kill("after-forward", step)
    opt.zero_grad()
    y.pow(2).mean().backward()
    opt.step()
    slots = [s for s in range(6) if (s + step) %% 3]
    append(slots, y.detach()[slots])
    kill("after-append", step)
    if step %% 5 == 1:
        pool.free([3, 5])
        pool.fork([1, 2], [3, 5])
    kill("after-fork", step)
    state.step(step + 1)
h = hashlib.sha256()
for t in model.state_dict().values():
    h.update(t.numpy().tobytes())
for slot in range(6):
    held = [int(p) for p in pool.table[slot] if p >= 0]
    tokens = kv[:, held].reshape(3, -1, 16)[:, :int(pool.lengths[slot])]
    h.update(tokens.contiguous().numpy().tobytes())
print("final", h.hexdigest(), pool.lengths.tolist(), masks.state_dict(), flush=True)
state.close()
'''


@pytest.fixture(scope="module")
def uninterrupted(tmp_path_factory):
    import os
    import subprocess
    import sys

    d = tmp_path_factory.mktemp("rank")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    script = RANK_LOOP % {"python": sys.executable, "root": root}
    (d / "loop.py").write_text(script)
    env = dict(os.environ, TPI_DATA_DIRECTORY=str(d))
    env.pop("TPI_EVENTS_FILE", None)
    res = subprocess.run([sys.executable, str(d / "loop.py")], env=env, capture_output=True,
                         text=True, timeout=300)
    assert res.returncode == 0, res.stderr
    return script, [line for line in res.stdout.splitlines() if line.startswith("final")][0]


@pytest.mark.parametrize("where", ["after-forward", "after-append", "after-fork"])
def test_a_preempted_rank_goes_on_with_its_masks_and_pages(tmp_path, uninterrupted, where):
    """A rank that trains with dropout and keeps a paged cache is preempted inside a step: its
    successor ends with the parameters and the cached tokens of an uninterrupted run."""
    from terraform_provider_iterative_amd import backends
    from terraform_provider_iterative_amd.models.cloud import Cloud, Credentials, NodeCredentials
    from terraform_provider_iterative_amd.models.values import Environment, Task, Variables
    from terraform_provider_iterative_amd.utils.identifier import new_deterministic_identifier

    script, final = uninterrupted
    cloud = Cloud(provider="local",
                  credentials=Credentials(node=NodeCredentials(state_root=str(tmp_path / "st"))))
    task = backends.new(cloud, new_deterministic_identifier("pages-" + where), Task(
        environment=Environment(script=script, timeout=300, variables=Variables(
            {"TPI_TASK": "true", "KILL_WHERE": where}))))
    task.create()
    status = task.wait(240)
    logs = task.logs()
    task.delete()
    assert status["succeeded"] == 1 and len(logs) == 2, (status, logs)
    assert "start 7 " in logs[1], logs
    assert final in logs[1], (final, logs)


def test_a_save_in_the_middle_of_a_step_leaves_the_pages(tmp_path, monkeypatch):
    from terraform_provider_iterative_amd.checkpoint import preemption

    kv = torch.ones(10, 4)
    pool = ops.PagePool([kv], 4, 3, 4)
    pool.extend([0, 1], [9, 3])
    pool.free([0])
    state = TrainingState(torch.nn.Linear(2, 2), path=str(tmp_path / "spill"), tile_bytes=4096,
                          paged={"kv": pool})
    before = pool.meta.clone()
    monkeypatch.setattr(preemption, "_mid_step", True)
    state.save({"step": 1})
    assert torch.equal(pool.meta, before) and kv.all()
    monkeypatch.setattr(preemption, "_mid_step", False)
    state.save({"step": 2})
    assert pool.table[1, 0] == 0 and not kv[1:].any()
    state.close()


def test_paged_caches_are_checked_when_the_state_is_built():
    with pytest.raises(ValueError, match="paged 'kv' is on"):
        pool = ops.PagePool([torch.zeros(4, 4)], 4, 1)
        TrainingState(torch.nn.Linear(2, 2, device="meta"), paged={"kv": pool}, device="meta")
