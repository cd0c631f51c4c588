"""Dropout from a counter-based generator; its mask is never stored.

Whether an element is kept depends on three things only: a seed, the number of the draw, and the
element's index in the whole tensor (the definition is in ``csrc/common/philox.h``).  So

* the backward pass draws the mask again instead of reading it back,
* a checkpoint carries two integers (:class:`MaskStream` is ``stateful`` for
  :class:`~..checkpoint.TrainingState`), and a resumed rank draws what the uninterrupted one
  would have,
* the masks do not depend on how many ranks share a tensor (``shard=``): a gang that resumes
  with another number of ranks goes on with the same masks.

Device tensors go through ``csrc/hip/dropout.hip``, host tensors through
``csrc/torchext/dropout.cpp``, which is also the autograd node; both give the same bits.
"""
from __future__ import annotations

import threading
from typing import Any, List, NamedTuple, Optional, Sequence, Tuple, Union

import torch

from ._loader import torch_ext, torch_hip

_TYPES = (torch.float32, torch.float16, torch.bfloat16)
_WHOLE = 1 << 32


class Draw(NamedTuple):
    """What names one mask: ``(seed, number)``, or with ``state`` (an int64 tensor ``[seed,
    number]`` on the operand's device) ``state``'s seed and ``number`` past ``state``'s, which are
    read when a kernel runs (a :class:`MaskStream` gives its draws a state that stays as it is)."""
    seed: int
    number: int
    state: Optional[torch.Tensor] = None


class MaskStream:
    """Hands out draw numbers, and is what a checkpoint carries of all masks::

        masks = MaskStream(seed=7)
        state = TrainingState(model, opt, path=spill, stateful={"masks": masks})
        y = dropout(x, 0.1, masks)

    Each :func:`dropout` given the stream takes the next number.  A block that is computed twice
    (activation checkpointing) has to draw the same masks both times: take ``masks.next()``
    outside it and pass that, or give the stream's contexts to the checkpoint::

        y = checkpoint(block, x, use_reentrant=False, context_fn=masks.checkpoint_contexts)

    Without either the second computation, which is a part of the backward pass, is refused.

    With ``device`` the seed and number are held there and read when a kernel runs, so that a
    captured graph draws new masks at every replay: call :meth:`advance` once per step, inside
    the capture, after the step's last draw.  A draw keeps its mask, also once the stream has
    advanced (a block that the backward pass computes again).  Without it a capture is refused,
    because every replay would repeat the captured masks; so are ``torch.jit.trace``, ``make_fx`` and
    ``torch.export`` (they record a draw that is given as numbers, ``torch.ops.tpi.dropout``).
    """

    def __init__(self, seed: int = 0, number: int = 0, device=None):
        _check_key(seed, number)
        self.seed, self.number = int(seed), int(number)
        self.state: Optional[torch.Tensor] = None
        if device is not None:
            self.state = torch.tensor([_signed(self.seed), self.number], dtype=torch.int64,
                                      device=device)
            self._ahead = 0
            self._copies: dict = {}
            self._replayed = False  # a graph or a recorded program advances the state by itself

    def _where(self) -> Tuple[int, int]:
        """The stream that a kernel would go to, and the capture (0: none)."""
        return torch_hip().stream_and_capture(self.state.device.index) if self.state.is_cuda else (0, 0)

    def _copy(self, recorded: int) -> torch.Tensor:
        """What this step's draws refer to: a copy of the state, which advancing does not change.  One
        for each stream and each captured graph that draws, ordered before what it draws; where the
        state may have moved between two draws, one for each."""
        where = self._where()
        keep = not recorded and (where[1] or not self._replayed)
        copy = self._copies.get(where) if keep else None
        if copy is None:
            copy = self.state + 0  # a kernel
            if keep and type(copy) is torch.Tensor:  # not a fake one
                self._copies[where] = copy
        return copy

    def checkpoint_contexts(self) -> Tuple["_Frame", "_Frame"]:
        """``context_fn`` of ``torch.utils.checkpoint.checkpoint(use_reentrant=False)``: the draws
        that the block takes are kept, and given again when the backward pass computes it again."""
        draws: List[Draw] = []
        return _Frame(self, draws, False), _Frame(self, draws, True)

    def next(self) -> Draw:
        """The stream's next draw (inside :meth:`checkpoint_contexts`' second context, the one that
        the first one's block took here)."""
        around = torch_ext().surroundings()
        uses = [use for use in _frames.uses if use.frame.stream is self] if _frames.uses else ()
        for i in reversed(range(len(uses))):
            if uses[i].frame.again:
                draw = uses[i].take()
                uses = uses[i + 1:]  # blocks inside the one that is computed again
                break
        else:
            if around & _IN_BACKWARD:
                raise RuntimeError(
                    "a block that the backward pass computes again would draw another mask: take its "
                    "draw outside (draw = masks.next()), or checkpoint it with "
                    "context_fn=masks.checkpoint_contexts")
            draw = self._next(around & _RECORDED)
        for use in uses:
            use.frame.draws.append(draw)
        return draw

    def _next(self, recorded: int) -> Draw:
        if self.state is not None:
            copy = self._copy(recorded)
            self._ahead += 1
            return Draw(0, self._ahead - 1, copy)
        if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            raise ValueError("a captured graph would repeat this stream's masks at every replay: "
                             "give MaskStream a device")
        if recorded:
            raise ValueError("a traced program would repeat this stream's mask at every run: "
                             "give dropout a draw of its own")
        self.number += 1
        return Draw(self.seed, self.number - 1)

    def advance(self) -> None:
        """End of a step (device streams): the next step's draws come after this one's."""
        if self.state is None:
            raise ValueError("advance() is for a MaskStream with a device")
        if self._where()[1] or torch_ext().surroundings() & _RECORDED:
            self._replayed = True
        self.state[1:].add_(self._ahead)
        self._ahead, self._copies = 0, {}

    def state_dict(self) -> dict:
        seed, number = self.seed, self.number
        if self.state is not None:
            seed, number = self.state.tolist()
            seed, number = seed % (1 << 64), number + self._ahead
        return {"seed": seed, "number": number}

    def load_state_dict(self, state: dict) -> None:
        seed, number = int(state["seed"]), int(state["number"])
        _check_key(seed, number)
        if self.state is not None:
            self.state.copy_(torch.tensor([_signed(seed), number], dtype=torch.int64))
            self._ahead, self._copies = 0, {}
        else:
            self.seed, self.number = seed, number


_IN_BACKWARD, _RECORDED = 1, 2  # torch_ext().surroundings()


class _Frames(threading.local):
    """The contexts that a thread is in, the innermost last."""

    def __init__(self):
        self.uses: List["_Use"] = []


_frames = _Frames()


class _Frame:
    """A block that may be computed twice: ``draws`` are what it has taken from ``stream`` the first
    time, and what it gets ``again``."""

    def __init__(self, stream: MaskStream, draws: List[Draw], again: bool):
        self.stream, self.draws, self.again = stream, draws, again

    def __enter__(self) -> "_Frame":
        if not self.again:
            self.draws.clear()
        _frames.uses.append(_Use(self))
        return self

    def __exit__(self, *exc: Any) -> None:
        last = max(i for i, use in enumerate(_frames.uses) if use.frame is self)
        del _frames.uses[last]


class _Use:
    """One pass through a frame's block: every backward pass over a graph makes one of its own."""

    def __init__(self, frame: _Frame):
        self.frame, self.given = frame, 0

    def take(self) -> Draw:
        draws = self.frame.draws
        if self.given == len(draws):
            raise RuntimeError("a block draws more masks when it is computed again (%d the first time)"
                               % len(draws))
        self.given += 1
        return draws[self.given - 1]


def _signed(value: int) -> int:
    return value - (1 << 64) if value >> 63 else value


def _check_key(seed, number) -> None:
    if not 0 <= seed < 1 << 64:
        raise ValueError("seed must be in [0, 2^64)")
    if not 0 <= number < 1 << 63:
        raise ValueError("draw number must be in [0, 2^63)")


def _as_draw(draw) -> Draw:
    if isinstance(draw, MaskStream):
        return draw.next()
    if not isinstance(draw, Draw):
        try:
            seed, number = draw
        except (TypeError, ValueError):
            raise TypeError("draw must be a MaskStream, a Draw or (seed, number)") from None
        draw = Draw(int(seed), int(number))
    _check_key(draw.seed, draw.number)
    if draw.state is not None and (draw.state.dtype != torch.int64 or draw.state.numel() != 2
                                   or not draw.state.is_contiguous()):
        raise ValueError("a draw's state must be two contiguous int64")
    return draw


def keep_threshold(p: float) -> Tuple[int, float]:
    """``(threshold, scale)`` of a drop probability: an element is kept when its 32-bit uniform
    number is below ``threshold``, and the scale is the inverse of the share that this keeps
    (``threshold / 2^32``), not of ``1 - p``, so that the expectation is exact."""
    p = float(p)
    if not 0.0 <= p <= 1.0:  # NaN too
        raise ValueError("dropout probability must be in [0, 1]")
    threshold = int(round((1.0 - p) * _WHOLE))
    return threshold, (_WHOLE / threshold if threshold else 0.0)


def _shard_walk(shape, shard) -> Tuple[int, List[int]]:
    """Index of a shard's first element in the whole tensor, and its index strides."""
    whole, starts = (tuple(int(v) for v in part) for part in shard)
    if len(whole) != len(shape) or len(starts) != len(shape):
        raise ValueError("shard must give a size and a start for each of the %d dimensions"
                         % len(shape))
    strides, step, first = [], 1, 0
    for size, lo, n in zip(reversed(whole), reversed(starts), reversed(shape)):
        if lo < 0 or lo + n > size:
            raise ValueError("shard %s at %s is not inside %s" % (tuple(shape), starts, whole))
        strides.append(step)
        first += lo * step
        step *= size
    if step >= 1 << 63:
        raise ValueError("the whole tensor is too large")
    return first, strides[::-1]


def dropout(x: torch.Tensor, p: float, draw: Union[MaskStream, Draw, Tuple[int, int]], *,
            residual: Optional[torch.Tensor] = None,
            shard: Optional[Tuple[Sequence[int], Sequence[int]]] = None) -> torch.Tensor:
    """``x`` with each element dropped with probability ``p`` and the others scaled by
    ``1 / (1 - p)``, plus ``residual``; differentiable in both.

    ``x`` is float32, float16 or bfloat16, on the GPU or the host, of any strides that merge into
    6 dimensions.  ``residual`` has its shape and device, and its type or float32; the result
    has the residual's type (computed in 32 bits, rounded once).  A dropped element contributes
    0 whatever ``x`` holds there.  ``p`` is taken to the nearest multiple of 2^-32.

    ``draw`` names the mask: a :class:`MaskStream` (its next number), or ``(seed, number)``,
    which gives the same mask at every call (and every replay of a captured one).
    ``shard=(whole_shape, starts)`` says that ``x`` is the block of a tensor of ``whole_shape``
    that begins at ``starts``: it is masked as that block of the whole would be.

    ``x`` and ``residual`` are strided tensors with memory of their own (of a DTensor, its local part
    with ``shard=``).  The result is enqueued on the current stream of ``x``'s device.
    """
    if not isinstance(x, torch.Tensor) or not (x.is_cuda or x.is_cpu):
        raise TypeError("dropout needs a tensor on the GPU or the host")
    if x.dtype not in _TYPES:
        raise TypeError("dropout of %s is not supported (float32, float16, bfloat16)" % x.dtype)
    threshold, scale = keep_threshold(p)
    if residual is not None:
        if not isinstance(residual, torch.Tensor) or residual.device != x.device:
            raise ValueError("the residual must be a tensor on %s" % x.device)
        if residual.shape != x.shape:  # a broadcast one: expand it, its gradient is summed there
            raise ValueError("the residual's shape %s is not x's %s (expand it first)"
                             % (tuple(residual.shape), tuple(x.shape)))
        if residual.dtype not in (x.dtype, torch.float32):
            raise TypeError("the residual must be %s or float32" % x.dtype)
    first, strides = (0, ()) if shard is None else _shard_walk(x.shape, shard)
    draw = _as_draw(draw)
    if draw.state is not None and draw.state.device != x.device:
        raise ValueError("the mask stream is on %s, the tensor on %s" % (draw.state.device,
                                                                         x.device))
    ext = torch_hip() if x.is_cuda else torch_ext()
    return ext.dropout(x, residual, threshold, scale, *draw, first, strides)


class CounterDropout(torch.nn.Module):
    """:func:`dropout` as a layer: ``layer(x)`` or ``layer(x, residual)``.  Layers of a model
    share one :class:`MaskStream`; in evaluation nothing is drawn or dropped.  ``draw`` takes the
    place of the stream's next one (a layer in a block that is computed twice)."""

    def __init__(self, p: float, stream: MaskStream):
        super().__init__()
        keep_threshold(p)
        self.p, self.stream = float(p), stream

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                draw: Union[Draw, Tuple[int, int], None] = None) -> torch.Tensor:
        if self.training:
            return dropout(x, self.p, self.stream if draw is None else draw, residual=residual)
        return x if residual is None else dropout(x, 0.0, (0, 0), residual=residual)

    def extra_repr(self) -> str:
        return "p=%g" % self.p
