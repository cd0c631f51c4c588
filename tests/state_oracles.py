"""Oracles of the operators on a rank's state, written from their definitions: Philox in Python
integers, a pool of pages as lists."""
import numpy as np


# -- dropout from a counter-based generator ------------------------------------------------------

def philox4x32(counter, key, rounds=10):
    """Philox4x32 (Salmon et al., SC 2011) in Python integers."""
    c, (k0, k1) = list(counter), key
    for _ in range(rounds):
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(q >> 32) ^ c[1] ^ k0, q & 0xFFFFFFFF, (p >> 32) ^ c[3] ^ k1, p & 0xFFFFFFFF]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return tuple(c)


def keep_mask(indexes, p, seed, number):
    """Which elements (indexes in the whole tensor) are kept."""
    threshold = int(round((1.0 - p) * 2 ** 32))
    cache = {}

    def half(block, level, lane):
        if (block, level) not in cache:
            cache[block, level] = philox4x32(
                (block & 0xFFFFFFFF, block >> 32, number & 0xFFFFFFFF, number >> 32 | level << 31),
                (seed & 0xFFFFFFFF, seed >> 32))
        return cache[block, level][lane // 2] >> 16 * (lane % 2) & 0xFFFF

    return [(half(n // 8, 0, n % 8) << 16 | half(n // 8, 1, n % 8)) < threshold for n in indexes]


def dropout_oracle(x, p, draw, residual=None):
    """(kept, result) in 64 bits."""
    import torch

    kept = torch.tensor(keep_mask(range(x.numel()), p, *draw)).reshape(x.shape)
    scale = 2 ** 32 / int(round((1.0 - p) * 2 ** 32))
    out = torch.where(kept, x.detach().cpu().double() * scale, 0.0)
    return kept, out if residual is None else out + residual.detach().cpu().double()


# -- pages of a paged cache ----------------------------------------------------------------------

class PoolOracle:
    """A pool in plain Python on host tensors: the definition of every operation."""

    def __init__(self, tensors, tokens, slots, width):
        self.tensors, self.tokens, self.slots, self.width = tensors, tokens, slots, width
        self.pages = tensors[0].shape[0]
        self.rows = [[] for _ in range(slots)]
        self.lengths = np.zeros(slots, np.int64)
        self.stale = set(range(self.pages))

    @property
    def refs(self):
        return np.bincount(np.array(sum(self.rows, []), np.int64), minlength=self.pages)

    @property
    def table(self):
        return np.array([row + [-1] * (self.width - len(row)) for row in self.rows])

    def free_count(self):
        return int((self.refs == 0).sum())

    def _need(self, length):
        return -(-int(length) // self.tokens)

    def copy(self, src, dst):
        for t in self.tensors:
            t[list(dst)] = t[list(src)].clone()
        refs = self.refs  # a free page that is written is not known to be zero any more
        self.stale |= {int(d) for s, d in zip(src, dst) if s != d and refs[d] == 0}

    def extend(self, slots, tokens):
        counts = [tokens] * len(slots) if isinstance(tokens, int) else tokens
        for s, more in zip(slots, counts):
            self.lengths[s] += more
            free = iter(np.nonzero(self.refs == 0)[0].tolist())
            while len(self.rows[s]) < self._need(self.lengths[s]):
                self.rows[s].append(next(free))

    def fork(self, src, dst):
        rows, lengths = [list(r) for r in self.rows], self.lengths.copy()  # before the call
        for s, d in zip(src, dst):
            self.rows[d], self.lengths[d] = list(rows[s]), lengths[s]
            if lengths[s] % self.tokens:
                self.rows[d].pop()
                page = int(np.nonzero(self.refs == 0)[0][0])
                self.copy([rows[s][-1]], [page])
                self.rows[d].append(page)

    def free(self, slots):
        before = self.refs > 0
        for s in slots:
            self.rows[s], self.lengths[s] = [], 0
        self.stale |= set(np.nonzero(before & (self.refs == 0))[0].tolist())

    def compact(self, clear=False):
        refs = self.refs
        live = int((refs > 0).sum())
        holes = [p for p in range(live) if refs[p] == 0]
        movers = [p for p in range(live, self.pages) if refs[p] > 0]
        self.copy(movers, holes)
        to = dict(zip(movers, holes))
        self.rows = [[to.get(p, p) for p in row] for row in self.rows]
        self.stale = {p for p in (self.stale | set(movers)) if p >= live}
        if clear:
            for t in self.tensors:
                t[sorted(self.stale)] = 0
            self.stale = set()

    def refusal(self, act, *args):
        """Why a call is refused (a part of the message), None if it is not."""
        if act == "extend":
            slots, tokens = args
            counts = [tokens] * len(slots) if isinstance(tokens, int) else tokens
            now = [int(self.lengths[s]) + c for s, c in zip(slots, counts)]
            if any(self._need(n) > self.width for n in now):
                return "longer than a row"
            take = sum(self._need(n) - len(self.rows[s]) for s, n in zip(slots, now))
            return "not enough free pages" if take > self.free_count() else None
        if act == "fork":
            src, dst = args
            if any(s == d or self.lengths[d] for s, d in zip(src, dst)):
                return "holds a sequence"
            take = sum(int(self.lengths[s] % self.tokens != 0) for s in src)
            return "not enough free pages" if take > self.free_count() else None
        return None

    def random_call(self, rng):
        act = rng.choice(["extend", "extend", "extend", "fork", "free", "compact", "copy"])
        count = int(rng.randint(0, self.slots + 1))
        slots = rng.permutation(self.slots)[:count].tolist()
        if act == "extend":
            if rng.rand() < 0.5:
                return act, (slots[:3], int(rng.randint(0, 2 * self.tokens + 2)))
            return act, (slots[:4], rng.randint(0, 3 * self.tokens + 1, len(slots[:4])).tolist())
        if act == "fork":
            empty = [s for s in range(self.slots) if not self.lengths[s]]
            rng.shuffle(empty)
            dst = empty[:int(rng.randint(0, 4))] if rng.rand() < 0.9 else slots[:1]
            return act, (rng.randint(0, self.slots, len(dst)).tolist(), dst)
        if act == "free":
            return act, (slots[:max(1, self.slots // 3)],)
        if act == "compact":
            return act, (bool(rng.randint(2)),)
        pages = rng.permutation(self.pages)
        n = int(rng.randint(0, self.pages // 2 + 1))
        return act, (pages[:n].tolist(), pages[n:2 * n].tolist())
