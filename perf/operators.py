"""Measured cases of the operators on a rank's state: dropout from a counter-based generator, and the
pages of a paged cache (copying, forking, freeing, compacting).

``run`` computes each in elementary torch operations while ``own`` is false and through
``terraform_provider_iterative_amd.ops`` while it is true, on the same inputs.
"""
import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MASK32 = 0xFFFFFFFF
# Philox4x32 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011):
# the two multipliers and the two key increments of the published definition.
MUL0, MUL1 = 0xD2511F53, 0xCD9E8D57
ADD0, ADD1 = 0x9E3779B9, 0xBB67AE85
ROUNDS = 10


def listed():
    # Dropout: a forward and a backward pass each.  Sizes of examples/train (hidden 2048, 4 x as
    # wide inside, 16 x 512 tokens) and of the small models that tests train.
    cases = [
        # a test-sized model, where the launch counts
        dict(name="dropout_small", op="dropout", batch=4, seq=32, cols=64, dtype="bf16", p=0.1,
             residual="same"),
        # the end of a block: residual + dropout(x)
        dict(name="dropout_block", op="dropout", batch=16, seq=512, cols=2048, dtype="bf16",
             p=0.1, residual="same"),
        # the wide activation inside a block, no residual: the largest
        dict(name="dropout_wide", op="dropout", batch=16, seq=512, cols=8192, dtype="bf16",
             p=0.2, residual="none"),
        # odd sizes, and a residual stream that is kept in 32 bits
        dict(name="dropout_odd", op="dropout", batch=7, seq=509, cols=2047, dtype="fp16", p=0.37,
             residual="fp32"),
        # a rank's columns of a wider tensor (a quarter of its 2048), masked as the whole would be
        dict(name="dropout_shard", op="dropout", batch=16, seq=512, cols=512, dtype="fp32",
             p=0.5, residual="none", shard=True),
        # Pages.  One page of one layer, where the launch counts
        dict(name="copy_one", op="copy", pools=2, pages=64, tokens=16, heads=2, dim=64, pairs=1),
        # a batch's pages copied in every layer's keys and values
        dict(name="copy_many", op="copy", pools=16, pages=4096, tokens=16, heads=8, dim=128,
             pairs=1024),
        # pages whose bytes are no multiple of any vector
        dict(name="copy_odd", op="copy", pools=6, pages=2000, tokens=13, heads=3, dim=37,
             pairs=777),
        # 32 prompts with 4 continuations each: full pages shared, the last one copied
        dict(name="fork_samples", op="fork", pools=8, pages=8192, tokens=16, heads=8, dim=128,
             slots=192, seqs=32, lo=5, hi=2003, fan=4, share=False),
        # what a scheduler does between two steps: sequences end, others branch, all grow by one
        dict(name="turnover", op="turnover", pools=16, pages=8192, tokens=16, heads=4, dim=128,
             slots=256, seqs=192, lo=17, hi=1000, fan=1, share=True),
        # live pages to the front of the pool, before a checkpoint
        dict(name="compact_half", op="compact", pools=16, pages=4096, tokens=16, heads=4, dim=128,
             slots=128, seqs=100, lo=40, hi=500, share=True, clear=False),
        # the same for a large pool whose dead pages are cleared as well: the largest
        dict(name="compact_clear", op="compact", pools=16, pages=8192, tokens=16, heads=8,
             dim=128, slots=300, seqs=256, lo=1, hi=600, share=True, clear=True),
    ]
    return cases


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["dropout", "dropout", "dropout", "copy", "fork", "turnover", "compact"])
    if op == "dropout":
        shard = rng.random() < 0.25
        cols = _log(rng, 40, 8192)
        rows = _log(rng, 1, max(2, min(16 * 512, (1 << 26) // cols)))
        batch = rng.choice([1, 2, 3, 5, 8])
        residual = "none" if shard else rng.choice(["none", "same", "fp32"])
        dtype = rng.choice(list(DTYPES))
        return dict(op=op, batch=batch, seq=max(1, rows // batch), cols=cols, dtype=dtype,
                    p=round(rng.uniform(0.01, 0.9), 4), residual=residual, shard=shard)
    shape = dict(op=op, pools=rng.choice([1, 2, 3, 8, 16]), tokens=rng.choice([1, 8, 13, 16, 32]),
                 heads=rng.choice([1, 2, 3, 4, 8]), dim=rng.choice([37, 64, 80, 128]))
    if op == "copy":
        pairs = _log(rng, 1, 1000)
        return dict(shape, pages=2 * pairs + rng.randint(0, 900), pairs=pairs)
    seqs, lo = _log(rng, 2, 128), rng.randint(1, 60)
    hi = lo + _log(rng, 1, 600) * shape["tokens"] // 16
    fan = rng.randint(1, 3) if op == "fork" else 1
    slots = seqs * (1 + fan) + rng.randint(0, 20)
    need = seqs * (-(-hi // shape["tokens"]) + 1 + fan) + 1
    case = dict(shape, pages=need + rng.randint(0, 1000), slots=slots, seqs=seqs, lo=lo, hi=hi,
                share=rng.random() < 0.5)
    if op == "compact":
        return dict(case, clear=rng.random() < 0.5)
    return dict(case, fan=fan)


# -- inputs ----------------------------------------------------------------------------------------

def _counts(case):
    """Sequence lengths, and for each sequence how many pages it has and shares with the sequence
    before it: fixed by the case, so that its work is known."""
    n, tokens = case["seqs"], case["tokens"]
    lengths = [case["lo"] + (case["hi"] - case["lo"]) * i // max(1, n - 1) for i in range(n)]
    pages = [-(-v // tokens) for v in lengths]
    shared = [lengths[i - 1] // tokens // 2 if case["share"] and i % 2 else 0 for i in range(n)]
    return lengths, pages, shared


def _turnover(case):
    """Sequence numbers that end, that branch, and how many go on."""
    n = case["seqs"]
    ends, branches = list(range(0, n, 4)), list(range(1, n, 4))
    return ends, branches


def _metadata(case, rng):
    """Table, lengths and reference counts of a fragmented pool, and each sequence's slot."""
    lengths, pages, shared = _counts(case)
    live = sum(pages) - sum(shared)
    total = case["pages"]
    moved = min(live, total - live) // 2 if live > 1 else 0
    ids = np.concatenate([rng.permutation(live)[:live - moved],
                          live + rng.permutation(total - live)[:moved]])
    rng.shuffle(ids)
    slot = rng.permutation(case["slots"])
    width = max(pages) + 2
    table = np.full((case["slots"], width), -1, np.int32)
    length = np.zeros(case["slots"], np.int32)
    refs = np.zeros(total, np.int32)
    at = 0
    for i in range(case["seqs"]):
        row = table[slot[i]]
        if shared[i]:
            row[:shared[i]] = table[slot[i - 1]][:shared[i]]
        fresh = pages[i] - shared[i]
        row[shared[i]:pages[i]] = ids[at:at + fresh]
        at += fresh
        length[slot[i]] = lengths[i]
        refs[row[:pages[i]]] += 1
    return table, length, refs, slot


def _pool(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    shape = (case["pools"], case["pages"], case["tokens"], case["heads"], case["dim"])
    kv = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    return kv.normal_(generator=g)


def prepare(case, seed):
    rng = np.random.RandomState(seed & 0x7FFFFFFF)
    if case["op"] == "dropout":
        g = torch.Generator("cuda").manual_seed(seed)
        shape = (case["batch"], case["seq"], case["cols"])
        dtype = DTYPES[case["dtype"]]

        def normal(kind):
            return torch.randn(shape, dtype=torch.float32, device="cuda", generator=g).to(kind)

        state = {"case": case, "x": normal(dtype).requires_grad_(True), "residual": None,
                 "key": int(rng.randint(1 << 62, dtype=np.int64)),
                 "draw": int(rng.randint(1 << 40, dtype=np.int64))}
        out = dtype
        if case["residual"] != "none":
            out = torch.float32 if case["residual"] == "fp32" else dtype
            state["residual"] = normal(out).requires_grad_(True)
        state["grad"] = normal(out)
        return state
    kv = _pool(case, seed)
    state = {"case": case, "kv": kv}
    dev = dict(dtype=torch.int32, device="cuda")
    if case["op"] == "copy":
        order = rng.permutation(case["pages"])
        n = case["pairs"]
        state["src"] = torch.tensor(order[:n], **dev)
        state["dst"] = torch.tensor(order[n:2 * n], **dev)
        if own:
            from terraform_provider_iterative_amd import ops

            state["pool"] = ops.PagePool(list(kv.unbind(0)), page_tokens=case["tokens"], slots=1)
        return state
    table, length, refs, slot = _metadata(case, rng)
    state["table"] = torch.tensor(table, **dev)
    state["lengths"] = torch.tensor(length, **dev)
    state["refs"] = torch.tensor(refs, **dev)
    n = case["seqs"]
    if case["op"] == "fork":
        state["src"] = torch.tensor(np.repeat(slot[:n], case["fan"]), **dev)
        state["dst"] = torch.tensor(slot[n:n + n * case["fan"]], **dev)
    elif case["op"] == "turnover":
        ends, branches = _turnover(case)
        gone = np.zeros(n, bool)
        gone[ends] = True
        state["end"] = torch.tensor(slot[ends], **dev)
        state["src"] = torch.tensor(slot[branches], **dev)
        state["dst"] = torch.tensor(slot[n:n + len(branches)], **dev)
        state["grow"] = torch.tensor(np.concatenate([slot[:n][~gone],
                                                     slot[n:n + len(branches)]]), **dev)
    if own:
        from terraform_provider_iterative_amd import ops

        state["pool"] = ops.PagePool(list(kv.unbind(0)), page_tokens=case["tokens"],
                                     slots=case["slots"], width=table.shape[1])
        state["pool"].bind(state["table"], state["lengths"])
        state["saved"] = state["pool"].meta.clone()
    return state


# -- dropout, plain --------------------------------------------------------------------------------

def _threshold(p):
    """Element kept if its 32-bit uniform number is below this; the share kept is exactly
    threshold / 2^32, and the scale is its inverse."""
    keep = int(round((1.0 - p) * 4294967296.0))
    return keep, float(np.float32(4294967296.0 / keep))


def _mul(m, x):
    """High and low 32 bits of a 32 x 32-bit product, in 64-bit integers without a sign."""
    t = m * (x & 0xFFFF)
    u = m * (x >> 16) + (t >> 16)
    return u >> 16, ((u & 0xFFFF) << 16) | (t & 0xFFFF)


def _philox(block, c2, c3, key):
    a, b = block & MASK32, block >> 32
    c, d = torch.full_like(block, c2), torch.full_like(block, c3)
    k0, k1 = key & MASK32, key >> 32
    for _ in range(ROUNDS):
        h0, l0 = _mul(MUL0, a)
        h1, l1 = _mul(MUL1, c)
        a, b, c, d = h1 ^ b ^ k0, l1, h0 ^ d ^ k1, l0
        k0, k1 = (k0 + ADD0) & MASK32, (k1 + ADD1) & MASK32
    return torch.stack([a & 0xFFFF, a >> 16, b & 0xFFFF, b >> 16,
                        c & 0xFFFF, c >> 16, d & 0xFFFF, d >> 16], dim=-1)


def _kept(case, key, number):
    """Truth value of every element.  Element n of the whole tensor has half-word n % 8 of block
    n / 8; the generator's first number gives the high half of its 32 bits, its second the low."""
    rows, cols = case["batch"] * case["seq"], case["cols"]
    first, step = _index(case)
    if step == cols and first % 8 == 0:  # one run of elements
        rows, cols, step = 1, rows * cols, 0
    start = first + step * torch.arange(rows, device="cuda")
    block = (start >> 3)[:, None] + torch.arange(-(-cols // 8) + 1, device="cuda")
    high = _philox(block, number & MASK32, number >> 32, key)
    low = _philox(block, number & MASK32, (number >> 32) | 0x80000000, key)
    number32 = ((high << 16) | low).flatten(1)
    if first % 8 or step % 8:
        at = (start & 7)[:, None] + torch.arange(cols, device="cuda")
        number32 = number32.gather(1, at)
    kept = number32[:, :cols] < _threshold(case["p"])[0]
    return kept.reshape(case["batch"], case["seq"], case["cols"])


def _index(case):
    """Index in the whole tensor of the first element, and from one row to the next."""
    if case.get("shard"):
        return 2 * case["cols"], 4 * case["cols"]
    return 0, case["cols"]


def _dropout(state):
    case, x, grad = state["case"], state["x"], state["grad"]
    scale = _threshold(case["p"])[1]
    kept = _kept(case, state["key"], state["draw"])
    zero = torch.zeros((), device="cuda")
    out = torch.where(kept, x.detach().float() * scale, zero)
    dx = torch.where(kept, grad.float() * scale, zero).to(x.dtype)
    if state["residual"] is None:
        return {"out": out.to(x.dtype), "dx": dx}
    residual = state["residual"].detach()
    return {"out": (out + residual.float()).to(residual.dtype), "dx": dx, "dresidual": grad}


def _own_dropout(state):
    from terraform_provider_iterative_amd import ops

    case, x, residual = state["case"], state["x"], state["residual"]
    shard = None
    if case.get("shard"):
        shard = ((case["batch"], case["seq"], 4 * case["cols"]), (0, 0, 2 * case["cols"]))
    out = ops.dropout(x, case["p"], (state["key"], state["draw"]), residual=residual, shard=shard)
    if residual is None:
        dx, = torch.autograd.grad(out, (x,), state["grad"])
        return {"out": out.detach(), "dx": dx}
    dx, dr = torch.autograd.grad(out, (x, residual), state["grad"])
    return {"out": out.detach(), "dx": dx, "dresidual": dr}


# -- pages, plain ----------------------------------------------------------------------------------

def _free(table, lengths, refs, slots, tokens):
    rows = table[slots]
    held = torch.arange(table.shape[1], device="cuda") < -(-lengths[slots] // tokens)[:, None]
    refs = refs.index_add(0, rows[held], torch.full((), -1, dtype=torch.int32,
                                                    device="cuda").expand(int(held.sum())))
    table = table.index_fill(0, slots.long(), -1)
    return table, lengths.index_fill(0, slots.long(), 0), refs


def _fork(kv, table, lengths, refs, src, dst, tokens):
    length = lengths[src]
    full = length // tokens
    at = torch.arange(table.shape[1], device="cuda")
    rows = torch.where(at < full[:, None], table[src], -1)
    held = rows[rows >= 0]
    refs = refs.index_add(0, held, torch.ones((), dtype=torch.int32,
                                              device="cuda").expand(held.numel()))
    part = (length % tokens != 0).nonzero().flatten()  # their last page is copied
    fresh = (refs == 0).nonzero().flatten()[:part.numel()]
    last = full[part].long()
    kv[:, fresh] = kv[:, table[src[part].long(), last].long()]
    rows[part, last] = fresh.int()
    refs[fresh] = 1
    return table.index_copy(0, dst.long(), rows), lengths.index_copy(0, dst.long(), length), refs


def _extend(table, lengths, refs, slots, more, tokens):
    length = lengths[slots]
    new = -(-(length + more) // tokens)
    at = torch.arange(table.shape[1], device="cuda")
    want = (at >= -(-length // tokens)[:, None]) & (at < new[:, None])
    row, column = want.nonzero(as_tuple=True)  # in the order of the slots asked for
    fresh = (refs == 0).nonzero().flatten()[:row.numel()]
    table = table.index_put((slots[row].long(), column), fresh.int())
    refs = refs.index_fill(0, fresh, 1)
    return table, lengths.index_copy(0, slots.long(), length + more), refs


def _compact(kv, table, refs, clear):
    live = refs > 0
    n = int(live.sum())
    holes = (~live[:n]).nonzero().flatten()
    moved = live[n:].nonzero().flatten() + n
    kv[:, holes] = kv[:, moved]
    to = torch.arange(refs.numel(), dtype=torch.int32, device="cuda")
    to[moved] = holes.int()
    table = torch.where(table >= 0, to[table.clamp(min=0).long()], table)
    refs = refs.index_copy(0, holes, refs[moved])
    refs[n:] = 0
    if clear:
        kv[:, n:] = 0
    return table, refs


def _pages(state):
    case, kv = state["case"], state["kv"]
    tokens = case["tokens"]
    if case["op"] == "copy":
        kv[:, state["dst"].long()] = kv[:, state["src"].long()]
        return {"kv": kv.view(torch.int16)}
    table, lengths, refs = state["table"], state["lengths"], state["refs"]
    if case["op"] == "turnover":
        table, lengths, refs = _free(table, lengths, refs, state["end"], tokens)
    if case["op"] in ("fork", "turnover"):
        table, lengths, refs = _fork(kv, table, lengths, refs, state["src"], state["dst"], tokens)
    if case["op"] == "turnover":
        table, lengths, refs = _extend(table, lengths, refs, state["grow"], 1, tokens)
    if case["op"] == "compact":
        table, refs = _compact(kv, table, refs, case["clear"])
    return {"kv": kv.view(torch.int16), "table": table, "lengths": lengths, "refs": refs}


def _own_pages(state):
    case, kv, pool = state["case"], state["kv"], state["pool"]
    if case["op"] == "copy":
        pool.copy(state["src"], state["dst"])
        return {"kv": kv.view(torch.int16)}
    pool.meta.copy_(state["saved"])  # every pass starts from the same pool
    if case["op"] == "turnover":
        pool.free(state["end"])
    if case["op"] in ("fork", "turnover"):
        pool.fork(state["src"], state["dst"])
    if case["op"] == "turnover":
        pool.extend(state["grow"], 1)
    if case["op"] == "compact":
        pool.compact(clear=case["clear"])
    return {"kv": kv.view(torch.int16), "table": pool.table, "lengths": pool.lengths,
            "refs": pool.refs}


def run(state):
    if state["case"]["op"] == "dropout":
        return _own_dropout(state) if own else _dropout(state)
    return _own_pages(state) if own else _pages(state)


# -- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    if case["op"] == "dropout":
        n = case["batch"] * case["seq"] * case["cols"]
        size = 4 if case["dtype"] == "fp32" else 2
        out = 4 if case["residual"] == "fp32" else size
        residual = out if case["residual"] != "none" else 0
        return {"bytes": n * (size + residual + out + out + size), "flops": 3 * n}
    page = 2 * case["tokens"] * case["heads"] * case["dim"] * case["pools"]
    if case["op"] == "copy":
        return {"bytes": case["pairs"] * (2 * page + 8), "flops": 0}
    lengths, pages, shared = _counts(case)
    tokens = case["tokens"]
    live = sum(pages) - sum(shared)
    if case["op"] == "compact":
        moved = min(live, case["pages"] - live) // 2 if live > 1 else 0
        # every page that moves; the table's held entries and the counts, read and written
        size = moved * 2 * page + 8 * sum(pages) + 8 * case["pages"]
        return {"bytes": size + (case["pages"] - live) * page * case["clear"], "flops": 0}
    size = 0
    branch = list(range(case["seqs"]))
    if case["op"] == "turnover":
        ends, branch = _turnover(case)
        size += sum(pages[i] for i in ends) * 12  # table entry cleared, count read and written
        size += (case["seqs"] - len(ends) + len(branch)) * 8  # lengths read and written
    for i in branch:  # table entries read and written, counts read and written, last page copied
        size += case["fan"] * (16 * pages[i] + (2 * page if lengths[i] % tokens else 0))
    return {"bytes": size, "flops": 0}


# -- the definition in 64 bits ---------------------------------------------------------------------

def _uniform16(n, level, key, number):
    """Half-word of each element index in ``n`` (numpy, 64 bits without a sign)."""
    u = np.uint64
    word = [n // u(8) & u(MASK32), n // u(8) >> u(32), u(number & MASK32),
            u((number >> 32) | level << 31)]
    keys = [key & MASK32, key >> 32]
    for _ in range(ROUNDS):
        p, q = word[0] * u(MUL0), word[2] * u(MUL1)
        word = [(q >> u(32)) ^ word[1] ^ u(keys[0]), q & u(MASK32),
                (p >> u(32)) ^ word[3] ^ u(keys[1]), p & u(MASK32)]
        keys = [(keys[0] + ADD0) & MASK32, (keys[1] + ADD1) & MASK32]
    return word


def _half(words, lane):
    """Half-words ``lane`` (0 to 7) of the four words of a block."""
    pick = np.choose(lane // 2, words)
    return (pick >> (np.uint64(16) * (lane % 2).astype(np.uint64))) & np.uint64(0xFFFF)


def exact(case, seed):
    if case["op"] != "dropout":
        return None  # pages are moved, nothing is computed
    state = prepare(case, seed)
    first, step = _index(case)
    rows, cols, keep = case["batch"] * case["seq"], case["cols"], _threshold(case["p"])[0]
    high, low = np.uint64(keep >> 16), np.uint64(keep & 0xFFFF)
    kept = np.empty((rows, cols), bool)
    per = max(1, (1 << 22) // cols)
    for r in range(0, rows, per):
        count = min(per, rows - r)
        n = (np.uint64(first) + np.uint64(step) * np.arange(r, r + count, dtype=np.uint64)[:, None]
             + np.arange(cols, dtype=np.uint64))
        block, where = np.unique(n >> np.uint64(3), return_inverse=True) if step % 8 or first % 8 \
            else (None, None)
        if block is None:  # whole blocks: row by row
            width = -(-cols // 8)
            starts = n[:, :1] + np.uint64(8) * np.arange(width, dtype=np.uint64)
            words = np.stack(_uniform16(starts, 0, state["key"], state["draw"])[0:4], axis=-1)
            top = words.astype("<u4").view("<u2").reshape(count, -1)[:, :cols]
        else:
            words = np.stack(_uniform16(block << np.uint64(3), 0, state["key"], state["draw"]),
                             axis=-1)
            halves = words.astype("<u4").view("<u2").reshape(-1, 8)
            top = halves[where.reshape(n.shape), (n & np.uint64(7)).astype(np.int64)]
        kept[r:r + count] = top < high
        ties = np.nonzero(top == high)
        at = n[ties]
        rest = _half(_uniform16(at, 1, state["key"], state["draw"]), (at % np.uint64(8)).astype(int))
        kept[r:r + count][ties] = rest < low
    mask = torch.from_numpy(kept).cuda().reshape(state["x"].shape)
    scale = 4294967296.0 / keep
    out = torch.where(mask, state["x"].detach().double() * scale, 0.0)
    dx = torch.where(mask, state["grad"].double() * scale, 0.0)
    if state["residual"] is None:
        return {"out": out, "dx": dx}
    return {"out": out + state["residual"].detach().double(), "dx": dx,
            "dresidual": state["grad"].double()}
