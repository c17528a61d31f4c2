"""The operators of the 4-bit key/value cache as workloads: inputs, plain forms, exact values and costs.

A cache row (the key or the value of one token and one head) is held in blocks of 32 values: 4-bit codes c, a step s (f16) and
a lowest value lo (bf16), x' = lo + s c.  Records of 32 tokens of one head lie in pages; a table names the pages of every sequence.

  store   quantises the new rows of a batch of sequences into their pages (and reads them back, which is its result)
  load    reads rows back as numbers
  attend  attention of the new rows over the cache, with the log of the sums and the attention each slot received
  evict   keeps the slots that received most attention, moves them to other pages (and reads them back)

`own` false: elementary torch operations on the same page bytes.  `own` true: the framework's operators.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
TILE = 32    # tokens of a record
BLOCK = 32   # values of a block


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one new token of one short conversation: latency is all there is
        dict(name="attend_first_tokens", op="attend", type="bf16", seqs=1, kv_heads=2, group=4, dim=64, page=32, length=33,
             rows=1, ragged=False, causal=True, window=0, weights=False),
        # a serving batch, one new token each, sequences of many lengths
        dict(name="attend_batch", op="attend", type="bf16", seqs=64, kv_heads=8, group=4, dim=128, page=64, length=8192,
             rows=1, ragged=True, causal=True, window=0, weights=False),
        # one long document, one new token: the axis of the slots has to be split
        dict(name="attend_long", op="attend", type="bf16", seqs=1, kv_heads=8, group=8, dim=128, page=256, length=131072,
             rows=1, ragged=False, causal=True, window=0, weights=False),
        # a batch that keeps book of the attention its slots receive, for the eviction to come
        dict(name="attend_counted", op="attend", type="f16", seqs=32, kv_heads=8, group=4, dim=128, page=64, length=4096,
             rows=1, ragged=True, causal=True, window=0, weights=True),
        # a part of a prompt that joins what the cache holds already
        dict(name="attend_prompt_part", op="attend", type="bf16", seqs=2, kv_heads=8, group=4, dim=128, page=64, length=10007,
             rows=2048, ragged=False, causal=True, window=0, weights=False),
        # a few proposed tokens to verify, single precision, a sliding window, odd counts
        dict(name="attend_proposed", op="attend", type="f32", seqs=9, kv_heads=3, group=5, dim=64, page=32, length=2777,
             rows=7, ragged=True, causal=True, window=1000, weights=True),
        # one new row a sequence
        dict(name="store_tokens", op="store", type="bf16", seqs=64, kv_heads=8, dim=128, page=64, length=4096, rows=1, ragged=True),
        # prompts of several sequences
        dict(name="store_prompts", op="store", type="bf16", seqs=5, kv_heads=8, dim=128, page=64, length=9001, rows=8192, ragged=True),
        # a short cache read back in single precision
        dict(name="load_small", op="load", type="f32", seqs=3, kv_heads=4, dim=64, page=32, length=701, rows=701, ragged=True),
        # a whole cache read back, to go elsewhere
        dict(name="load_all", op="load", type="bf16", seqs=8, kv_heads=8, dim=128, page=64, length=16384, rows=16384, ragged=True),
        # a conversation that has outgrown its budget by a little
        dict(name="evict_small", op="evict", type="bf16", seqs=2, kv_heads=4, dim=64, page=32, length=1100, keep=1001, first=4, recent=256),
        # a batch of long sequences cut to a quarter
        dict(name="evict_batch", op="evict", type="bf16", seqs=16, kv_heads=8, dim=128, page=64, length=16384, keep=4096, first=4,
             recent=1024),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "store", "load", "evict"])
    c = dict(op=op, type=rng.choice(["bf16", "bf16", "f16", "f32"]), seqs=_log(rng, 1, 64), kv_heads=rng.choice([1, 2, 3, 4, 5, 8]),
             dim=rng.choice([64, 128, 128, 256]), page=rng.choice([32, 64, 128, 256]))
    values = c["seqs"] * c["kv_heads"] * c["dim"]
    c["length"] = _log(rng, 16, max(16, min(131072, 2 ** 28 // values)))
    if op == "attend":
        c["group"] = rng.choice([1, 2, 3, 4, 5, 8, 16])
        kind = rng.choice(["token", "token", "few", "part"])
        most = {"token": 1, "few": 16, "part": 2048}[kind]
        pairs = 2 ** 37 // (values * c["length"] * c["group"])
        c["rows"] = min(_log(rng, 1, most), c["length"], max(1, pairs))
        c["causal"] = rng.random() < 0.8
        c["window"] = rng.choice([0, 0, 0, _log(rng, 1, c["length"])])
        c["weights"] = rng.random() < 0.3
    elif op == "evict":
        c["length"] = max(c["length"], 32)
        c["keep"] = _log(rng, 8, c["length"])
        c["first"] = rng.randint(0, min(8, c["keep"] // 4))
        c["recent"] = rng.randint(0, c["keep"] // 2)
        return c
    else:
        c["rows"] = c["length"] if op == "load" else min(_log(rng, 1, 8192), c["length"])
    c["ragged"] = rng.random() < 0.7
    return c


def _counts(case):
    """Lengths of the sequences and the new rows of each: part of the case, not of the seed."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    lengths, rows = [], []
    for i in range(case["seqs"]):
        n = case["length"] if i == 0 or not case.get("ragged", True) else max(1, int(case["length"] * rng.uniform(0.1, 1.0)))
        r = case.get("rows", n)
        lengths.append(n)
        rows.append(min(n, r if i == 0 or not case.get("ragged", True) or r == case.get("length") else rng.randint(1, r)))
    return lengths, rows


# ------------------------------------------------------------------------------------------------ the format
def _below(lo):
    """The next bf16 below."""
    i = lo.view(torch.int16)
    return torch.where(lo > 0, i - 1, torch.where(lo < 0, i + 1, -32767)).to(torch.int16).view(torch.bfloat16)


def _above(s):
    """The next f16 above, of a number that is not negative."""
    return (s.view(torch.int16) + 1).to(torch.int16).view(torch.float16)


def _quantise(x):
    """x [..., d] -> (codes int64 [..., d], step f16 [..., d/32], lowest bf16 [..., d/32]), decided in 64 bits."""
    b = x.double().unflatten(-1, (-1, BLOCK))
    low = b.amin(-1)
    lo = low.to(torch.float32).to(torch.bfloat16)
    lo = torch.where(lo.double() > low, _below(lo), lo)
    need = (b.amax(-1) - lo.double()) / 15.0
    s = need.to(torch.float32).to(torch.float16)
    s = torch.where(s.double() < need, _above(s), s)
    s64, lo64 = s.double()[..., None], lo.double()[..., None]
    at = torch.where(s64 > 0, (b - lo64) / s64, 0.0)
    c = torch.floor(at + 0.5).clamp(0, 15)
    # next to a border the quotient may have been rounded across it; the border itself is exact in 64 bits
    c = torch.where((c < 15) & (s64 > 0) & (b >= lo64 + (c + 0.5) * s64), c + 1, c)
    c = torch.where((c > 0) & (b < lo64 + (c - 0.5) * s64), c - 1, c)
    return c.long().flatten(-2), s, lo


def _record_bytes(d):
    return TILE * (d + 8 * (d // BLOCK))


def _pack(k, v):
    """Rows [..., 32 tokens, d] -> records [..., bytes]."""
    d = k.shape[-1]
    nb, lead = d // BLOCK, k.shape[:-2]
    ck, sk, lk = _quantise(k)
    cv, sv, lv = _quantise(v)
    n = len(lead)
    # keys: token, then group g of 8 values of a block, then block: values 32 b + 8 g + 2 p + h in a word's bits 4 p + 16 h
    a = ck.reshape(*lead, 32, nb, 4, 2, 2, 2).permute(*range(n), n, n + 2, n + 1, n + 5, n + 3, n + 4)
    a = (a[..., 0] | (a[..., 1] << 4)).to(torch.uint8).reshape(*lead, -1)
    # values: eight tokens, then 16 i + m, then token: value 64 i + 16 p + m in a halfword's bits 4 p
    e = cv.reshape(*lead, 4, 8, d // 64, 2, 2, 16).permute(*range(n), n, n + 2, n + 5, n + 1, n + 3, n + 4)
    e = (e[..., 0] | (e[..., 1] << 4)).to(torch.uint8).reshape(*lead, -1)
    by_octet = lambda t: t.reshape(*lead, 4, 8, nb).transpose(-1, -2).contiguous().reshape(*lead, -1).view(torch.uint8)
    return torch.cat([a, e, by_octet(sk), by_octet(sv), lk.contiguous().reshape(*lead, -1).view(torch.uint8), by_octet(lv)], -1)


def _unpack(rec, d):
    """Records [..., bytes] -> K, V [..., 32, d] in 32 bits."""
    nb, lead, n = d // BLOCK, rec.shape[:-1], rec.dim() - 1
    half, side = 16 * d, 64 * nb
    parts = torch.split(rec, [half, half, side, side, side, side], -1)
    nibbles = lambda x: torch.stack([x & 15, x >> 4], -1)
    a = nibbles(parts[0]).reshape(*lead, 32, 4, nb, 2, 2, 2).permute(*range(n), n, n + 2, n + 1, n + 4, n + 5, n + 3)
    e = nibbles(parts[1]).reshape(*lead, 4, d // 64, 16, 8, 2, 2).permute(*range(n), n, n + 3, n + 1, n + 4, n + 5, n + 2)
    ck = a.reshape(*lead, 32, nb, BLOCK).float()
    cv = e.reshape(*lead, 32, nb, BLOCK).float()
    f16 = lambda x: x.contiguous().view(torch.float16).float()
    bf16 = lambda x: x.contiguous().view(torch.bfloat16).float()
    tokens = lambda t: t.reshape(*lead, 4, nb, 8).transpose(-1, -2).reshape(*lead, 32, nb, 1)
    sk, sv, lk, lv = tokens(f16(parts[2])), tokens(f16(parts[3])), bf16(parts[4]).reshape(*lead, 32, nb, 1), tokens(bf16(parts[5]))
    return (lk + sk * ck).flatten(-2), (lv + sv * cv).flatten(-2)


# ------------------------------------------------------------------------------------------------ inputs
def _rows_like_keys(shape, g, dtype):
    """Rows with channels of their own means, a few of them large, as keys have."""
    d = shape[-1]
    mean = torch.randn(shape[-2] if len(shape) > 2 else 1, d, generator=g, device="cuda")
    mean = mean * torch.where(torch.rand(mean.shape, generator=g, device="cuda") < 0.05, 4.0, 0.4)
    return (torch.randn(shape, generator=g, device="cuda") * 0.8 + mean).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)
    op, d, h, page, seqs = case["op"], case["dim"], case["kv_heads"], case["page"], case["seqs"]
    dtype = TYPES[case["type"]]
    lengths, rows = _counts(case)
    per_seq = -(-max(lengths) // page)
    used = [-(-n // page) for n in lengths]
    n_pages = sum(used) + 3
    pool = n_pages + (sum(-(-min(n, case["keep"]) // page) for n in lengths) if op == "evict" else 0)
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)

    def table_of(counts, width, skip):
        at = torch.tensor([0] + counts[:-1], device="cuda").cumsum(0)[:, None] + torch.arange(width, device="cuda") + skip
        there = torch.arange(width, device="cuda") < torch.tensor(counts, device="cuda")[:, None]
        return torch.where(there, order[at.clamp(max=pool - 1)], 0).to(torch.int32)

    st = dict(case=dict(case), seqs=seqs, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
              starts=torch.tensor([0] + rows, device="cuda").cumsum(0).to(torch.int32), total=sum(rows), max_rows=max(rows),
              max_length=max(lengths), table=table_of(used, per_seq, 0))
    if op == "store":
        st["pages"] = torch.zeros(pool, h, page // TILE, _record_bytes(d), dtype=torch.uint8, device="cuda")
        st["k"] = _rows_like_keys((st["total"], h, d), g, dtype)
        st["v"] = torch.randn(st["total"], h, d, generator=g, device="cuda").to(dtype)
    else:
        # what the pages hold was stored earlier: every record is filled, whether a sequence owns it or not
        st["pages"] = torch.cat([_pack(_rows_like_keys((n, page // TILE, TILE, h, d), g, dtype).permute(0, 3, 1, 2, 4),
                                       torch.randn(n, h, page // TILE, TILE, d, generator=g, device="cuda").to(dtype))
                                 for n in [min(1024, pool - i) for i in range(0, pool, 1024)]])
    if op == "attend":
        st["q"] = (torch.randn(st["total"], h * case["group"], d, generator=g, device="cuda") * 1.2).to(dtype)
        st["out"] = torch.empty_like(st["q"])
        st["lse"] = torch.empty(st["total"], h * case["group"], device="cuda")
        if case["weights"]:
            st["prior"] = torch.rand(seqs, h, max(lengths), generator=g, device="cuda") ** 4
            st["weights"] = torch.zeros(seqs, h, max(lengths), device="cuda")
    elif op == "evict":
        keep = case["keep"]
        # attention received: most slots hardly any, some none at all (equal weights), a few a lot
        w = torch.rand(seqs, h, max(lengths), generator=g, device="cuda") ** 6 * 3
        st["weights"] = torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.2, 0.0, w)
        counts = [min(n, keep) for n in lengths]
        st["to_table"] = table_of([-(-n // page) for n in counts], -(-keep // page), n_pages)
        st["to_lengths"] = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        st["to_weights"] = torch.empty(seqs, h, keep, device="cuda")
        st["kept"] = torch.empty(seqs, h, keep, dtype=torch.int32, device="cuda")
        st["starts"] = torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)
        st["total"] = sum(counts)
    if op != "attend":
        st["k_out"] = torch.empty(st["total"], h, d, dtype=dtype, device="cuda")
        st["v_out"] = torch.empty_like(st["k_out"])
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(st):
    if own:
        return _own(st)
    return {"store": _plain_store, "load": _plain_load, "attend": _plain_attend, "evict": _plain_evict}[st["case"]["op"]](st)


def _own(st):
    c = st["case"]
    if "cache" not in st:   # the handle that a program makes once for its pages
        import importlib

        import __graft_entry__ as entry

        entry.load_package()
        cache4 = importlib.import_module("tirocinio_triennale_amd.cache")
        st["cache"] = cache4.Cache(st["pages"], c["kv_heads"], c["dim"], c["page"])
    cache = st["cache"]
    if c["op"] == "store":
        cache.store(st["k"], st["v"], st["table"], st["lengths"], st["starts"])
        cache.load(st["k_out"], st["v_out"], st["table"], st["lengths"], st["starts"])
        return st["k_out"], st["v_out"]
    if c["op"] == "load":
        cache.load(st["k_out"], st["v_out"], st["table"], st["lengths"], st["starts"])
        return st["k_out"], st["v_out"]
    if c["op"] == "attend":
        counted = dict(weights=st["weights"], prior=st["prior"]) if c["weights"] else {}
        cache.attend(st["q"], st["out"], st["table"], st["lengths"], st["starts"], causal=c["causal"], window=c["window"],
                     max_rows=st["max_rows"], max_length=st["max_length"], lse=st["lse"], **counted)
        return (st["out"], st["lse"], st["weights"]) if c["weights"] else (st["out"], st["lse"])
    cache.evict(st["weights"], st["table"], st["lengths"], c["keep"], st["to_table"], st["to_lengths"], first=c["first"],
                recent=c["recent"], max_length=st["max_length"], to_weights=st["to_weights"], kept=st["kept"])
    cache.load(st["k_out"], st["v_out"], st["to_table"], st["to_lengths"], st["starts"])
    return st["kept"], st["to_weights"], st["to_lengths"], st["k_out"], st["v_out"]


def _plain_rows(st, table):
    """All slots of all sequences, K and V [seqs, heads, slots, d] in 32 bits."""
    rec = st["pages"][table.long()].transpose(1, 2)
    k, v = _unpack(rec, st["case"]["dim"])
    return k.flatten(2, 4), v.flatten(2, 4)


def _of_packed(st, lengths, starts):
    """For every packed row: its sequence and its slot."""
    r = torch.arange(st["total"], device="cuda")
    s = torch.searchsorted(starts[1:].long().contiguous(), r, right=True)
    return s, r - starts.long()[s + 1] + lengths.long()[s]


def _plain_store(st):
    dtype = TYPES[st["case"]["type"]]
    outs = []
    for x in (st["k"], st["v"]):
        c, s, lo = _quantise(x)
        c = c.float().unflatten(-1, (-1, BLOCK))
        outs.append((lo.float()[..., None] + s.float()[..., None] * c).flatten(-2).to(dtype))
    return tuple(outs)


def _plain_load(st):
    dtype = TYPES[st["case"]["type"]]
    k, v = _plain_rows(st, st["table"])
    s, slot = _of_packed(st, st["lengths"], st["starts"])
    return k[s, :, slot].to(dtype), v[s, :, slot].to(dtype)


def _seen(c, lengths, rows, i, slots):
    """Which slots row i (of `rows`) of a sequence sees: [seqs, rows, slots]."""
    length = lengths.long()[:, None, None]
    at = length - rows[:, None, None] + i[None, :, None]
    j = slots[None, None, :]
    see = (j <= at) & (j < length) if c["causal"] else (j < length).expand(-1, i.numel(), -1)
    if c["window"]:
        see = see & (j > at - c["window"])
    return see & (i[None, :, None] < rows[:, None, None])


def _plain_attend(st):
    c = st["case"]
    h, group, d, most = c["kv_heads"], c["group"], c["dim"], st["max_rows"]
    k, v = _plain_rows(st, st["table"])
    starts = st["starts"].long()
    rows = starts[1:] - starts[:-1]
    i = torch.arange(most, device="cuda")
    at = (starts[:-1, None] + i).clamp(max=st["total"] - 1)
    q = st["q"][at].float().reshape(-1, most, h, group, d).permute(0, 2, 3, 1, 4).reshape(-1, h, group * most, d)
    see = _seen(c, st["lengths"], rows, i, torch.arange(k.shape[2], device="cuda"))[:, None, None]
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(d ** -0.5).unflatten(2, (group, most))
    s = s.masked_fill_(~see, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (top + total.log()).squeeze(-1)
    p = p.div_(torch.where(total == 0, 1.0, total))
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (group, most))
    there = i < rows[:, None]
    out = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[there].to(TYPES[c["type"]])
    lse = lse.permute(0, 3, 1, 2).flatten(2, 3)[there]
    if not c["weights"]:
        return out, lse
    held = torch.arange(st["max_length"], device="cuda") < st["lengths"][:, None, None]
    w = p.sum((2, 3))[..., :st["max_length"]]
    return out, lse, torch.where(held, st["prior"] + w, 0.0)


def _plain_evict(st):
    c = st["case"]
    keep, w, dtype = c["keep"], st["weights"], TYPES[c["type"]]
    length = st["lengths"].long()[:, None, None]
    j = torch.arange(w.shape[-1], device="cuda")
    rank = torch.where((j < c["first"]) | (j >= length - c["recent"]), math.inf, w)
    rank = torch.where(j < length, rank, -math.inf)
    best = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    if best.shape[-1] < keep:
        best = torch.cat([best, best.new_zeros(*best.shape[:2], keep - best.shape[-1])], -1)
    i = torch.arange(keep, device="cuda")
    there = i < length.clamp(max=keep)
    kept = torch.where(there, best, w.shape[-1]).sort(-1).values
    slot = torch.where(there, kept, 0)
    to_weights = torch.where(there, torch.gather(w, 2, slot), 0.0)
    k, v = _plain_rows(st, st["table"])
    take = lambda x: torch.gather(x, 2, slot[..., None].expand(-1, -1, -1, x.shape[-1])).transpose(1, 2)[there[:, 0]].to(dtype)
    return (torch.where(there, kept, -1).to(torch.int32), to_weights, length[:, 0, 0].clamp(max=keep).to(torch.int32), take(k), take(v))


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["type"]]
    lengths, rows = _counts(case)
    h, d = case["kv_heads"], case["dim"]
    slot = 5 * d / 4   # bytes of one slot and head: key and value
    if case["op"] in ("store", "load"):
        moved = sum(rows) * h
        # a store's rows are read, written in 4 bits, and what they became is written out; a load reads and writes
        return {"bytes": moved * (slot + 2 * d * size * (2 if case["op"] == "store" else 1)), "flops": moved * 2 * d * 4}
    if case["op"] == "evict":
        moved = sum(min(n, case["keep"]) for n in lengths) * h
        return {"bytes": sum(lengths) * h * 4 + moved * (2 * slot + 8 + 2 * d * size), "flops": sum(lengths) * h * 4}
    heads, bytes_, pairs = h * case["group"], 0, 0
    for n, r in zip(lengths, rows):
        first = max(0, n - r + 1 - case["window"]) if case["window"] else 0
        bytes_ += (n - first) * h * slot + (8 * n * h if case["weights"] else 0)
        for i in range(r):
            at = n - r + i
            pairs += (at + 1 if case["causal"] else n) - (max(0, at + 1 - case["window"]) if case["window"] else 0)
    bytes_ += sum(rows) * heads * (2 * d * size + 4)
    return {"bytes": bytes_, "flops": 4 * d * heads * pairs}


# ------------------------------------------------------------------------------------------------ in 64 bits, from the definition
def _value(st, table, seq, head, slot, which):
    """The numbers that slots stand for (seq, head, slot: index tensors of one shape): [..., d] in 64 bits, one byte
    address a value from the layout's definition."""
    c = st["case"]
    d, page = c["dim"], c["page"]
    nb = d // BLOCK
    flat = st["pages"].reshape(-1)
    rec_bytes = _record_bytes(d)
    p = table.long()[seq, slot // page]
    rec = ((p * c["kv_heads"] + head) * (page // TILE) + slot % page // TILE) * rec_bytes
    t = (slot % TILE)[..., None]
    j = torch.arange(d, device="cuda")
    b, r = j // 32, j % 32
    if which == "k":
        bit = 4 * (r % 8 // 2) + 16 * (r % 2)
        at = t * (d // 2) + (r // 8) * (4 * nb) + 4 * b + bit // 8
        shift = bit % 8
    else:
        bit = 4 * (j % 64 // 16)
        at = 16 * d + (t // 8) * (4 * d) + (j // 64 * 16 + j % 16) * 16 + (t % 8) * 2 + bit // 8
        shift = bit % 8
    code = (flat[rec[..., None] + at].long() >> shift) & 15
    sides = 32 * d
    blocks = torch.arange(nb, device="cuda")
    by_octet = ((t // 8) * nb + blocks) * 16 + (t % 8) * 2
    s_at = rec[..., None] + sides + (0 if which == "k" else 64 * nb) + by_octet
    lo_at = rec[..., None] + sides + 128 * nb + ((t * nb + blocks) * 2 if which == "k" else 64 * nb + by_octet)
    word = lambda a: (flat[a].int() | (flat[a + 1].int() << 8)).to(torch.int16)
    s, lo = word(s_at).view(torch.float16).double(), word(lo_at).view(torch.bfloat16).double()
    return lo.repeat_interleave(BLOCK, -1) + s.repeat_interleave(BLOCK, -1) * code


def _count_thresholds(x):
    b = x.double().unflatten(-1, (-1, BLOCK))
    low, high = b.min(-1).values, b.max(-1).values
    lo = low.to(torch.bfloat16)
    lo = torch.where(lo.double() > low, _below(lo), lo)
    s = ((high - lo.double()) / 15).to(torch.float16)
    s = torch.where(15 * s.double() < high - lo.double(), _above(s), s)
    lo, s = lo.double()[..., None], s.double()[..., None]
    c = sum((b >= lo + (j + 0.5) * s).double() for j in range(15))
    return (lo + s * torch.where(s > 0, c, 0.0)).flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    c, (lengths, rows) = st["case"], _counts(case)
    h = c["kv_heads"]
    heads = torch.arange(h, device="cuda")
    if c["op"] == "store":
        return _count_thresholds(st["k"]), _count_thresholds(st["v"])
    if c["op"] in ("load", "evict"):
        outs = {"k": [], "v": []}
        kept_all, weights_all = [], []
        for s, n in enumerate(lengths):
            if c["op"] == "load":
                slot = torch.arange(n - rows[s], n, device="cuda")[:, None].expand(-1, h)
            else:
                take = []
                for head in range(h):
                    w = st["weights"][s, head, :n].double()
                    if n > c["keep"]:
                        w[:c["first"]] = 1e300
                        w[n - c["recent"]:] = 1e300
                        # equal weights: the earlier slot
                        order = torch.argsort(-w, stable=True)[:c["keep"]]
                        take.append(order.sort().values)
                    else:
                        take.append(torch.arange(n, device="cuda"))
                slot = torch.stack(take, -1)
                kept = torch.full((h, c["keep"]), -1, dtype=torch.int32, device="cuda")
                kept[:, :slot.shape[0]] = slot.t().int()
                weight = torch.zeros(h, c["keep"], dtype=torch.float64, device="cuda")
                weight[:, :slot.shape[0]] = torch.gather(st["weights"][s].double(), 1, slot.t())
                kept_all.append(kept)
                weights_all.append(weight)
            for which in "kv":
                outs[which].append(_value(st, st["table"], torch.full_like(slot, s), heads.expand_as(slot), slot, which))
        k, v = torch.cat(outs["k"]), torch.cat(outs["v"])
        if c["op"] == "load":
            return k, v
        to_lengths = torch.tensor([min(n, c["keep"]) for n in lengths], dtype=torch.int32, device="cuda")
        return torch.stack(kept_all), torch.stack(weights_all), to_lengths, k, v
    if 4 * c["dim"] * h * c["group"] * sum(n * r for n, r in zip(lengths, rows)) > 2e13:
        return None
    group, d = c["group"], c["dim"]
    out = torch.zeros(st["total"], h * group, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(st["total"], h * group, dtype=torch.float64, device="cuda")
    weights = torch.zeros(len(lengths), h, st["max_length"], dtype=torch.float64, device="cuda")
    first = 0
    for s, (n, r) in enumerate(zip(lengths, rows)):
        slot = torch.arange(n, device="cuda")
        see = torch.ones(r, n, dtype=torch.bool, device="cuda")
        i = torch.arange(r, device="cuda")[:, None] + (n - r)
        if c["causal"]:
            see &= slot <= i
        if c["window"]:
            see &= slot > i - c["window"]
        for head in range(h):
            seq, hd = torch.full_like(slot, s), torch.full_like(slot, head)
            k, v = (_value(st, st["table"], seq, hd, slot, which) for which in "kv")
            if c["weights"]:
                weights[s, head, :n] = st["prior"][s, head, :n].double()
            for j in range(group):
                q = st["q"][first:first + r, head * group + j].double()
                a = (q @ k.t()) / math.sqrt(d)
                a[~see] = -math.inf
                z = torch.logsumexp(a, -1)
                p = torch.where(see, (a - z[:, None]).exp(), 0.0)
                out[first:first + r, head * group + j] = p @ v
                lse[first:first + r, head * group + j] = z
                if c["weights"]:
                    weights[s, head, :n] += p.sum(0)
        first += r
    return (out, lse, weights) if c["weights"] else (out, lse)
