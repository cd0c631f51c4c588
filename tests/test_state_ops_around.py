"""Operators on a rank's state (tests/test_state_ops.py) where they meet what surrounds them:
checkpoints, other tensors than plain ones, transformations of a program."""
import pytest
import torch
import torch.distributed as dist

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
