"""Plain-Python reference implementations the native/HIP data plane is checked against."""
from __future__ import annotations

import struct

import numpy as np
import xxhash

POLY = 0x82F63B78
_TABLE = []
for _v in range(256):
    _c = _v
    for _ in range(8):
        _c = (_c >> 1) ^ POLY if _c & 1 else _c >> 1
    _TABLE.append(_c)


def crc32c_py(data: bytes, crc: int = 0) -> int:
    crc ^= 0xFFFFFFFF
    for byte in data:
        crc = (crc >> 8) ^ _TABLE[(crc ^ byte) & 0xFF]
    return crc ^ 0xFFFFFFFF


def crc32c_np(data: bytes) -> int:
    """Byte-serial CRC32C in numpy-free Python but tolerable for a few hundred KB."""
    return crc32c_py(data)


def shard_hash_py(data: bytes, shard_bytes: int = 1 << 20, seed: int = 0):
    """Striped-XXH64 shard digests (definition in csrc/common/xxh64.h)."""
    out = []
    for base in range(0, len(data), shard_bytes):
        d = data[base:base + shard_bytes]
        nstripes = (len(d) + 31) // 32
        digests = []
        for lane in range(256):
            msg = b"".join(d[32 * s:32 * s + 32] for s in range(lane, nstripes, 256))
            digests.append(xxhash.xxh64(msg, seed=seed).intdigest())
        out.append(xxhash.xxh64(struct.pack("<256Q", *digests), seed=seed).intdigest())
    return np.array(out, dtype=np.uint64)


def _a16(x: int) -> int:
    return (x + 15) & ~15


def _huf_plane_py(blob: bytes, off: int, n: int, ngroups: int, m: int, nesc: int,
                  dictionary: np.ndarray) -> np.ndarray:
    """HUF plane: canonical Huffman over dictionary + escape (symbol m, then 8 raw bits),
    LSB-first bits, substream s = groups s, s+256, ... (spec: csrc/common/tpz.h)."""
    streams = min(256, ngroups)
    lens = list(blob[off:off + 16])
    ends = [int(x) for x in np.frombuffer(blob, np.uint32, streams, off + 16)]
    base = off + 16 + _a16(4 * streams)
    table = {}  # (length, MSB-first code) -> symbol
    code = 0
    for length in range(1, 12):
        for s in range(m + 1):
            if lens[s] == length:
                table[(length, code)] = s
                code += 1
        code <<= 1
    vals = np.zeros(n, np.uint8)
    start = 0
    for s in range(streams):
        raw = np.frombuffer(blob, np.uint8, 4 * (ends[s] - start), base + 4 * start)
        bits = np.unpackbits(raw, bitorder="little").tolist() + [0] * 32
        pos = 0
        for g in range(s, ngroups, 256):
            for i in range(g * 32, min(g * 32 + 32, n)):
                c, length = 0, 0
                while (length, c) not in table:
                    c = (c << 1) | bits[pos]
                    pos += 1
                    length += 1
                    assert length <= 11, "no code"
                sym = table[(length, c)]
                if sym == m:
                    vals[i] = sum(bits[pos + b] << b for b in range(8))
                    pos += 8
                else:
                    vals[i] = dictionary[sym]
        assert pos <= 32 * (ends[s] - start)
        start = ends[s]
    assert start == nesc
    return vals


def tpz_decode_tile_py(blob: bytes, length: int) -> np.ndarray:
    """Independent numpy decoder of one TPZ1 tile blob (spec: csrc/common/tpz.h)."""
    n = length // 4
    ngroups = (n + 31) // 32
    out = np.zeros(length, np.uint8)
    off = 96
    for p in range(4):
        k, m, _, _, nesc = struct.unpack_from("<BBBBI", blob, 24 * p)
        dictionary = np.frombuffer(blob, np.uint8, 16, 24 * p + 8)
        if k == 8:  # raw plane
            out[p::4] = np.frombuffer(blob, np.uint8, n, off)
            off += ngroups * 32
            continue
        if k == 9:  # Huffman plane
            out[p::4] = _huf_plane_py(blob, off, n, ngroups, m, nesc, dictionary)
            off += 16 + _a16(4 * min(256, ngroups)) + _a16(4 * nesc)
            continue
        if k == 0:  # constant plane
            out[p::4] = dictionary[0]
            continue
        esc_code = (1 << k) - 1
        words = np.frombuffer(blob, np.uint32, ngroups * k, off)
        bits = np.unpackbits(words.view(np.uint8), bitorder="little")
        codes = bits[:ngroups * 32 * k].reshape(-1, k).astype(np.uint32)
        codes = (codes << np.arange(k, dtype=np.uint32)).sum(axis=1)[:n]
        escapes = np.frombuffer(blob, np.uint8, nesc, off + _a16(ngroups * 4 * k))
        vals = dictionary[np.minimum(codes, m - 1)].copy()
        is_esc = codes == esc_code
        assert int(is_esc.sum()) == nesc
        vals[is_esc] = escapes
        out[p::4] = vals
        off += _a16(ngroups * 4 * k) + _a16(nesc)
    return out


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
