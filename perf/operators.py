"""Measured cases of the request-batch operators: block tables, the paged 8-bit K/V cache (append and attention) and sampling.

A decode server's step over this library runs them in this order: finished requests give their blocks back and the
others get blocks, slots and positions for their new tokens (tables), the new K/V rows enter the 8-bit pools (append),
every row attends its own request (attend), and the logits become tokens (sample).  Shapes are those of the
repository's models (32/8 and 64/8 heads of 128, 32/4 heads of 64, vocabularies of 128256 and 32000, contexts of 8192).
"""
import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}  # the library's activation dtype codes
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
POOL = {"i8": (torch.int8, 127.0, 0), "e4m3": (torch.float8_e4m3fn, 448.0, 1)}  # torch type, largest value, library code


# ---- cases ------------------------------------------------------------------------------------------------------------

def tables(n_seq, max_len, chunk, block, tight):
    return {"op": "tables", "n_seq": n_seq, "max_len": max_len, "chunk": chunk, "block": block, "tight": tight}


def append(n_seq, tokens, kv_heads, head_dim, block, pool, dtype):
    return {"op": "append", "n_seq": n_seq, "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim, "block": block,
            "pool": pool, "dtype": dtype}


def attend(n_seq, min_len, max_len, rows, heads, kv_heads, head_dim, block, pool, dtype):
    return {"op": "attend", "n_seq": n_seq, "min_len": min_len, "max_len": max_len, "rows": rows, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "block": block, "pool": pool, "dtype": dtype}


def sample(rows, vocab, dtype, temperature, top_k, top_p, min_p, spread):
    return {"op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": temperature, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "spread": spread}


def listed():
    return [
        # one decode step of a small server: a token per request, some requests finished
        dict(tables(64, 8192, 1, 16, False), name="tables 64 decode"),
        # a large server admitting prompts beside its decodes, short of blocks for the last of them
        dict(tables(1024, 4096, 500, 32, True), name="tables 1024 mixed"),
        # the K/V rows of a decode step: one token a request, most blocks part filled
        dict(append(32, 1, 8, 128, 16, "i8", "f32"), name="append 32 decode"),
        # prompts of some hundred tokens each, activations in 16 bits
        dict(append(9, 700, 8, 128, 64, "e4m3", "bf16"), name="append 6300 prompt"),
        # a single stream in a short context: latency
        dict(attend(1, 777, 777, 1, 32, 8, 128, 16, "i8", "f32"), name="attend 1 x 777"),
        # a single stream at the 70B shape's context
        dict(attend(1, 8192, 8192, 1, 64, 8, 128, 16, "i8", "f32"), name="attend 1 x 8192"),
        # a ragged decode batch
        dict(attend(32, 1, 8192, 1, 64, 8, 128, 16, "i8", "f32"), name="attend 32 ragged"),
        # four draft rows a request of a small model, checked in one call
        dict(attend(64, 100, 1999, 4, 32, 4, 64, 32, "e4m3", "f16"), name="attend 64 x 4 rows"),
        # long contexts
        dict(attend(16, 30000, 65536, 1, 64, 8, 128, 64, "e4m3", "bf16"), name="attend 16 long"),
        # one stream's next token with the usual chat settings
        dict(sample(1, 128256, "f32", 0.8, 40, 0.95, 0.05, 2.5), name="sample 1"),
        # a batch whose requests each have settings of their own
        dict(sample(64, 128256, "f32", 1.0, -1, -1.0, -1.0, 2.5), name="sample 64 mixed"),
        # a wide batch of a small vocabulary, temperature and nucleus alone, 16-bit logits
        dict(sample(333, 32000, "bf16", 0.7, 0, 0.9, 0.0, 2.0), name="sample 333 nucleus"),
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    op = rng.choice(["tables", "append", "attend", "attend", "sample", "sample"])
    block = rng.choice([16, 32, 64, 128])
    pool, dtype = rng.choice(["i8", "e4m3"]), rng.choice(["f32", "f16", "bf16"])
    heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (64, 8, 128), (32, 4, 64), (16, 16, 64), (8, 1, 128), (24, 2, 128)])
    if op == "tables":
        return tables(log(1, 1024), log(1, 8192), rng.choice([1, log(1, 500)]), block, rng.random() < 0.5)
    if op == "append":
        tokens = rng.choice([1, log(1, 700)])
        return append(log(1, max(1, 6000 // tokens)), tokens, kv_heads, head_dim, block, pool, dtype)
    if op == "attend":
        top = log(1, 65536)
        n_seq = log(1, max(1, min(256, 16 * 40000 // max(top, 64))))
        rows = rng.choice([1, 1, 1, 2, 5]) if top <= 2048 else 1
        n_seq = max(1, n_seq // rows)
        return attend(n_seq, max(1, min(top, log(1, top))), top, rows, heads, kv_heads, head_dim, block, pool, dtype)
    vocab = log(300, 200000)
    rows = log(1, max(1, min(512, 64 * 128256 // vocab)))
    if rng.random() < 0.4:
        return sample(rows, vocab, dtype, 1.0, -1, -1.0, -1.0, rng.uniform(0.5, 4.0))
    return sample(rows, vocab, dtype, rng.choice([0.0, rng.uniform(0.2, 1.5)]), rng.choice([0, 1, log(2, 2000)]),
                  rng.choice([1.0, rng.uniform(0.1, 0.99)]), rng.choice([0.0, rng.uniform(0.001, 0.3)]), rng.uniform(0.5, 4.0))


def lengths(n, lo, hi):
    """n lengths from lo to hi, spread evenly and out of order; the first is hi."""
    return [hi - int((hi - lo + 1) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]


def blocks_of(tokens, block):
    return -(-tokens // block)


def table_sizes(case):
    """(have, done, add, table stride, blocks, rows) of a tables case: plain numbers, the same for every seed."""
    n, block = case["n_seq"], case["block"]
    have = [h if i % 16 else 0 for i, h in enumerate(lengths(n, 0, case["max_len"]), 1)]
    done = [i % 7 == 3 for i in range(n)]
    add = [0 if done[i] or i % 11 == 5 else case["chunk"] - i % 3 if case["chunk"] > 8 and i % 8 == 2 else 1 for i in range(n)]
    stride = blocks_of(case["max_len"] + case["chunk"], block)
    held = sum(blocks_of(h, block) for h in have)
    freed = sum(blocks_of(h, block) for h, d in zip(have, done) if d)
    need = sum(blocks_of(h + a, block) - blocks_of(h, block) for h, a in zip(have, add))
    spare = max(0, need - freed) + 64
    if case["tight"]:
        spare = max(1, need * 3 // 4 - freed)
    return have, done, add, stride, held + spare, blocks_of(sum(add) + 1, 64) * 64


def append_sizes(case):
    """(positions held, positions added) of every request of an append case."""
    n, tokens = case["n_seq"], case["tokens"]
    have = lengths(n, 0, 4 * case["block"]) if tokens == 1 else [h if i % 2 else 0 for i, h in enumerate(lengths(n, 0, 2 * case["block"]))]
    return have, lengths(n, -(-tokens // 2), tokens)


def work(case):
    op = case["op"]
    if op == "tables":
        have, done, add, stride, _, rows = table_sizes(case)
        block = case["block"]
        moved = sum(blocks_of(h, block) for h, d in zip(have, done) if d)
        new = sum(blocks_of(h + a, block) - blocks_of(h, block) for h, a in zip(have, add))
        return {"bytes": 4 * (6 * case["n_seq"] + 3 * rows + 2 * moved + 2 * new + 8), "flops": 0}
    kvd = case.get("kv_heads", 0) * case.get("head_dim", 0)
    if op == "append":
        have, add = append_sizes(case)
        block, new = case["block"], sum(add)
        back = sum(h + a - h // block * block for h, a in zip(have, add))  # tokens of the touched blocks, read back
        touched = sum(blocks_of(h + a, block) - h // block for h, a in zip(have, add))
        return {"bytes": 2 * kvd * (new * (SIZE[case["dtype"]] + 1) + back * 5) + touched * case["kv_heads"] * 16 + 4 * (new + back),
                "flops": 6 * kvd * new}
    if op == "attend":
        lens = lengths(case["n_seq"], case["min_len"], case["max_len"])
        rows, heads, hd = case["rows"], case["heads"], case["head_dim"]
        seen = sum(max(0, n - j) for n in lens for j in range(rows))
        pages = sum(blocks_of(n, case["block"]) for n in lens)
        return {"bytes": 2 * kvd * sum(lens) + pages * (8 * case["kv_heads"] + 4) + 2 * len(lens) * rows * heads * hd * SIZE[case["dtype"]],
                "flops": 4 * hd * heads * seen}
    return {"bytes": case["rows"] * (case["vocab"] * SIZE[case["dtype"]] + 28), "flops": 4 * case["rows"] * case["vocab"]}


# ---- inputs -----------------------------------------------------------------------------------------------------------

def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def quantised(gen, blocks, kv_heads, block, head_dim, pool):
    """A pool of filled blocks and its scales: normal values with a few strong channels, as keys have them."""
    kind, top, _ = POOL[pool]
    gain = torch.exp(0.4 * torch.randn(kv_heads, 1, head_dim, device=DEV, generator=gen))
    x = torch.randn(blocks, kv_heads, block, head_dim, device=DEV, generator=gen).mul_(gain)
    scale = x.abs().amax((2, 3)) / top
    x.div_(scale[:, :, None, None])
    q = x.round_().clamp_(-top, top).to(kind) if pool == "i8" else x.to(kind)
    return q, scale


def paged(case, gen, lens, spare):
    """Pools, scales and the block table of requests that hold `lens` tokens; `spare` more blocks are on no request."""
    block = case["block"]
    counts = [blocks_of(n, block) for n in lens]
    blocks, stride = sum(counts) + spare, max(1, max(counts))
    perm = torch.randperm(blocks, device=DEV, generator=gen, dtype=torch.int32)
    table = torch.zeros(len(lens), stride, dtype=torch.int32, device=DEV)
    held = torch.arange(stride, device=DEV)[None] < torch.tensor(counts, device=DEV)[:, None]
    table[held] = perm[: sum(counts)]
    s = {"case": case, "table": table, "blocks": blocks, "stride": stride}
    for name in ("k", "v"):
        s[name], s[name + "_scale"] = quantised(gen, blocks, case["kv_heads"], block, case["head_dim"], case["pool"])
    return s


def slots_at(table, block, places):
    """Slots of (request, first position, count) runs under a block table."""
    seq = torch.tensor([r for r, _, n in places for _ in range(n)], dtype=torch.int64, device=DEV)
    pos = torch.tensor([p + i for _, p, n in places for i in range(n)], dtype=torch.int64, device=DEV)
    return (table[seq, pos // block].long() * block + pos % block).int()


def prepare(case, seed):
    gen = torch.Generator(DEV).manual_seed(seed)
    op = case["op"]
    if op == "tables":
        have, done, add, stride, blocks, rows = table_sizes(case)
        n, block = case["n_seq"], case["block"]
        counts = torch.tensor([blocks_of(h, block) for h in have], device=DEV)
        perm = torch.randperm(blocks, device=DEV, generator=gen, dtype=torch.int32)
        total = int(counts.sum())
        table = torch.zeros(n, stride, dtype=torch.int32, device=DEV)
        table[torch.arange(stride, device=DEV)[None] < counts[:, None]] = perm[:total]
        free = torch.zeros(blocks, dtype=torch.int32, device=DEV)
        free[: blocks - total] = perm[total:]
        return {"case": case, "have": ints(have), "done": ints([int(d) for d in done]), "add": ints(add), "table": table,
                "free": free, "n_free": ints([blocks - total]), "blocks": blocks, "stride": stride, "rows": rows,
                "kept": ints([0] * n), "height": ints([0]), "lens": ints([0] * n), "counts": ints([0] * 3),
                "last": ints([0] * n), "row": [ints([0] * rows) for _ in range(3)]}
    if op == "append":
        have, add = append_sizes(case)
        block, kvd = case["block"], case["kv_heads"] * case["head_dim"]
        s = paged(case, gen, [h + a for h, a in zip(have, add)], 8)
        places = [(r, h, a) for r, (h, a) in enumerate(zip(have, add))]
        s["slots"] = torch.cat([slots_at(s["table"], block, places), ints([-1] * 3)])  # a batch padded by three rows
        s["read"] = slots_at(s["table"], block, [(r, h // block * block, h + a - h // block * block) for r, h, a in places])
        n = s["slots"].numel()
        # now and then a token is larger than what its block has seen
        gain = torch.exp(0.5 * torch.randn(n, 1, device=DEV, generator=gen))
        for name in ("k_new", "v_new"):
            s[name] = (torch.randn(n, kvd, device=DEV, generator=gen) * gain).to(DTYPES[case["dtype"]])
        for name in ("k_out", "v_out"):
            s[name] = torch.empty(s["read"].numel(), kvd, device=DEV)
        return s
    if op == "attend":
        lens = lengths(case["n_seq"], case["min_len"], case["max_len"])
        rows, hd = case["rows"], case["head_dim"]
        s = paged(case, gen, lens, 8)
        s["seq"] = ints([r for r in range(len(lens)) for _ in range(rows)])
        s["pos"] = ints([n - rows + j for n in lens for j in range(rows)])  # a draft row before the first position: none to see
        s["q"] = (1.5 * torch.randn(len(lens) * rows, case["heads"] * hd, device=DEV, generator=gen)).to(DTYPES[case["dtype"]])
        s["out"] = torch.empty_like(s["q"])
        s["scale"] = 1.0 / math.sqrt(hd)
        return s
    rows, vocab = case["rows"], case["vocab"]
    z = case["spread"] * torch.randn(rows, vocab, device=DEV, generator=gen)
    z[:, ::1013] += 3.0 * case["spread"]  # the few tokens that a model favours
    z[:, 7::97] = -math.inf  # banned tokens
    uniform = torch.rand(4, rows, device=DEV, generator=gen)

    def setting(name, mixed):
        return mixed if case["top_p"] < 0 else torch.full((rows,), float(case[name]), device=DEV)

    odd = torch.arange(rows, device=DEV)
    return {"case": case, "logits": z.to(DTYPES[case["dtype"]]), "u": torch.rand(rows, device=DEV, generator=gen),
            "temperature": setting("temperature", torch.where(odd % 8 == 0, 0.0, 0.3 + uniform[0])),
            "top_k": setting("top_k", torch.where(odd % 3 == 0, 0.0, (uniform[1] * 200).floor())).int(),
            "top_p": setting("top_p", torch.where(odd % 4 == 1, 1.0, 0.5 + 0.5 * uniform[2])),
            "min_p": setting("min_p", torch.where(odd % 5 == 2, 0.0, 0.1 * uniform[3])),
            "ids": torch.empty(rows, dtype=torch.int32, device=DEV), "prob": torch.empty(rows, device=DEV)}


# ---- one pass ---------------------------------------------------------------------------------------------------------

def run(s):
    return {"tables": run_tables, "append": run_append, "attend": run_attend, "sample": run_sample}[s["case"]["op"]](s)


_context = []


def context():
    from shukuchi_b200 import cuda as sc
    if not _context:
        _context.append(sc.Context(0))
    return _context[0]


def pages(s):
    """The pools' handle, kept as a program keeps it."""
    from shukuchi_b200 import cuda as sc
    if "pages" not in s:
        c = s["case"]
        s["pages"] = sc.Pages(context(), s["k"].data_ptr(), s["v"].data_ptr(), s["k_scale"].data_ptr(), s["v_scale"].data_ptr(),
                              POOL[c["pool"]][2], s["blocks"], c["kv_heads"], c["head_dim"], c["block"])
    return s["pages"]


def run_tables(s):
    c = s["case"]
    block, stride, blocks, rows, n = c["block"], s["stride"], s["blocks"], s["rows"], c["n_seq"]
    if own:
        ctx, p = context(), torch.Tensor.data_ptr
        ctx.pages_release(n, block, blocks, stride, p(s["table"]), p(s["done"]), p(s["have"]), p(s["kept"]), p(s["free"]),
                          p(s["n_free"]), p(s["height"]))
        ctx.pages_assign(n, block, blocks, stride, rows, p(s["kept"]), p(s["add"]), p(s["table"]), p(s["free"]), p(s["height"]),
                         p(s["lens"]), p(s["counts"]), p(s["row"][0]), p(s["row"][1]), p(s["row"][2]), p(s["last"]))
        return {"kept": s["kept"], "free": s["free"], "height": s["height"], "table": s["table"], "lens": s["lens"],
                "counts": s["counts"], "slots": s["row"][0], "pos": s["row"][1], "seq": s["row"][2], "last": s["last"]}
    have, add, done, table = s["have"].long(), s["add"].long(), s["done"] != 0, s["table"].long()
    col = torch.arange(stride, device=DEV)
    # release: blocks of the finished requests on top of the free stack, in request order
    count = torch.where(done, (have + block - 1) // block, 0)
    first = count.cumsum(0) - count
    at = torch.where(col < count[:, None], s["n_free"].long() + first[:, None] + col, blocks)
    free = torch.cat([s["free"].long(), table.new_zeros(1)]).scatter(0, at.flatten(), table.flatten())[:blocks]
    height = s["n_free"].long() + count.sum()
    kept = torch.where(done, 0, have)
    # assign: rows and blocks in request order
    row_end = add.cumsum(0)
    ok = (kept + add <= stride * block) & ((add == 0) | (row_end <= rows))
    held = (kept + block - 1) // block
    need = torch.where(ok, (kept + add + block - 1) // block - held, 0)
    end = need.cumsum(0)
    ok = ok & ((need == 0) | (end <= height))
    lens = torch.where(ok, kept + add, kept)
    new = torch.where(ok, need, 0)
    j = col - held[:, None]
    fresh = (j >= 0) & (j < new[:, None])
    table = torch.where(fresh, free[(height - 1 - ((end - need)[:, None] + j)).clamp(0, blocks - 1)], table)
    r = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(row_end, r, right=True).clamp(max=n - 1)
    i = r - (row_end - add)[seq]
    live = (r < row_end[-1]) & ok[seq]
    pos = torch.where(live, kept[seq] + i, -1)
    slots = torch.where(live, table[seq, pos.clamp(min=0) // block] * block + pos % block, -1)
    counts = torch.stack([height[0] - new.sum(), live.sum(), (~ok).sum()])
    last = torch.where(ok & (add > 0), row_end - 1, -1)
    out = {"kept": kept, "free": free, "height": height, "table": table, "lens": lens, "counts": counts, "slots": slots,
           "pos": pos, "seq": torch.where(live, seq, -1), "last": last}
    return {k: v.int() for k, v in out.items()}


def run_append(s):
    c = s["case"]
    block, kv_heads, hd = c["block"], c["kv_heads"], c["head_dim"]
    kind, top, _ = POOL[c["pool"]]
    if own:
        p, g = torch.Tensor.data_ptr, pages(s)
        g.append(s["slots"].numel(), p(s["k_new"]), p(s["v_new"]), p(s["slots"]), dtype=GGML[c["dtype"]])
        g.read(s["read"].numel(), p(s["read"]), p(s["k_out"]), p(s["v_out"]))
        return {"k": s["k_out"], "v": s["v_out"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    # which row of the call a slot of the pool takes, if any; padding rows go to a slot behind the pool
    size = s["blocks"] * block
    count = s["slots"].numel()
    slot = torch.where(s["slots"] >= 0, s["slots"], size).long()
    taken = torch.full((size + 1,), -1, device=DEV).scatter(0, slot, torch.arange(count, device=DEV))[:size].view(-1, block)
    first = torch.where(taken >= 0, torch.arange(block, device=DEV), block).amin(1)  # the first offset that a block takes
    touched = (first < block)[:, None]
    held = (torch.arange(block, device=DEV) < first[:, None]) & touched
    largest = torch.full((1,), top, device=DEV)  # a tensor: a quotient by a plain number is a product with its reciprocal
    read = s["read"].long()
    out = {}

    def rounded(x):
        return x.round().clamp(-top, top).to(kind) if kind is torch.int8 else x.clamp(-top, top).to(kind)

    def one(name):
        x = s[name + "_new"].float().view(count, kv_heads, hd)
        x = torch.where((taken >= 0)[..., None, None], x[taken.clamp(min=0)], 0.0).transpose(1, 2)  # as the pool lies
        scale = s[name + "_scale"]
        old = torch.where((first == 0)[:, None], 0.0, scale)
        new = torch.where(touched, torch.maximum(old, x.abs().amax((2, 3)) / largest), scale)
        grown = rounded(s[name].float() * torch.where(new > old, old / new, 1.0)[..., None, None])
        fresh = rounded(torch.where(new[..., None, None] > 0, x / new[..., None, None], 0.0))
        value = torch.where(held[:, None, :, None], grown.float(), s[name].float())
        value = torch.where((taken >= 0)[:, None, :, None], fresh.float(), value)
        s[name].copy_(value)
        scale.copy_(new)
        out[name] = (value[read // block, :, read % block] * new[read // block][:, :, None]).view(-1, kv_heads * hd)
        out[name + "_scale"] = scale

    one("k")
    one("v")
    return out


def run_attend(s):
    c = s["case"]
    block, heads, kv_heads, hd = c["block"], c["heads"], c["kv_heads"], c["head_dim"]
    rows = s["q"].shape[0]
    if own:
        from shukuchi_b200 import cuda as sc
        p = torch.Tensor.data_ptr
        if "ws" not in s:
            s["ws"] = torch.empty(sc.pages_attend_ws(rows, heads, kv_heads, hd), dtype=torch.uint8, device=DEV)
        pages(s).attend(rows, p(s["q"]), p(s["out"]), heads, p(s["pos"]), p(s["table"]), s["stride"], c["n_seq"], s["scale"],
                        p(s["ws"]), s["ws"].numel(), row_seq=p(s["seq"]), dtype=GGML[c["dtype"]])
        return s["out"]
    group, n_seq, length = heads // kv_heads, c["n_seq"], s["stride"] * block
    at = s["table"].long()

    def gathered(name):  # [sequence][KV head][position][head_dim]
        x = s[name][at].float().mul_(s[name + "_scale"][at][..., None, None])
        return x.transpose(1, 2).reshape(n_seq, kv_heads, length, hd)

    # a row's head h reads KV head h % kv_heads
    q = s["q"].float().view(n_seq, c["rows"], group, kv_heads, hd).permute(0, 3, 1, 2, 4).reshape(n_seq, kv_heads, -1, hd)
    seen = torch.arange(length, device=DEV) <= s["pos"].view(n_seq, c["rows"])[..., None]
    seen = seen[:, None, :, None].expand(-1, kv_heads, -1, group, -1).reshape(n_seq, kv_heads, -1, length)
    score = torch.where(seen, (q @ gathered("k").transpose(2, 3)) * s["scale"], -math.inf)
    peak = score.amax(3, keepdim=True)
    weight = torch.where(seen, torch.exp(score - torch.where(peak > -math.inf, peak, 0.0)), 0.0)
    total = weight.sum(3, keepdim=True)
    out = (weight @ gathered("v")) / torch.where(total > 0, total, 1.0)
    out = out.view(n_seq, kv_heads, c["rows"], group, hd).permute(0, 2, 3, 1, 4).reshape(rows, heads * hd)
    return out.to(s["q"].dtype)


def run_sample(s):
    c = s["case"]
    if own:
        p = torch.Tensor.data_ptr
        context().sample(p(s["logits"]), c["rows"], c["vocab"], p(s["u"]), p(s["ids"]), prob=p(s["prob"]),
                         temperature=p(s["temperature"]), top_k=p(s["top_k"]), top_p=p(s["top_p"]), min_p=p(s["min_p"]),
                         dtype=GGML[c["dtype"]])
        return {"ids": s["ids"], "prob": s["prob"]}
    z, index = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)
    t = s["temperature"][:, None]
    x = (z - z[:, :1]) * (1.0 / t)
    w = torch.where(z == z[:, :1], 1.0, torch.where(x <= 0, torch.exp(x), 0.0))
    w = torch.where(t > 0, w, (torch.arange(c["vocab"], device=DEV) == 0).float())  # no temperature: the first of the largest
    # probabilities as whole numbers of 2^-40: a draw next to a border goes by sums that are exact in any order
    mass = (w.double() * 2.0**40).floor().long()
    k = s["top_k"][:, None].long()
    mass = torch.where((k <= 0) | (torch.arange(c["vocab"], device=DEV) < k), mass, 0)
    before = mass.cumsum(1) - mass
    need = torch.ceil(s["top_p"][:, None].double() * mass.sum(1, keepdim=True).double()).long().clamp(min=1)
    mass = torch.where((s["top_p"][:, None] >= 1) | (before < need), mass, 0)
    mass = torch.where((w >= s["min_p"][:, None]) | (w == 1), mass, 0)
    mass = torch.zeros_like(mass).scatter(1, index, mass)  # in the vocabulary's order
    ends = mass.cumsum(1)
    total = ends[:, -1:]
    at = torch.minimum((s["u"][:, None].double() * total.double()).floor().long(), total - 1)
    ids = (ends <= at).sum(1, keepdim=True)
    prob = (mass.gather(1, ids).double() / total.double()).float()
    return {"ids": ids[:, 0].int(), "prob": prob[:, 0]}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "append":
        return exact_append(s)
    if case["op"] == "attend":
        return exact_attend(s)
    return {"ids": None, "prob": exact_prob(s)}


def exact_append(s):
    """Block by block.  A block's scale is stored in 32 bits and the quotients are rounded to 32 bits before they are
    rounded to 8: both belong to the format."""
    c = s["case"]
    block, kv_heads, hd = c["block"], c["kv_heads"], c["head_dim"]
    kind, top, _ = POOL[c["pool"]]
    slots = s["slots"].tolist()
    runs = {}
    for t, slot in enumerate(slots):
        if slot >= 0:
            runs.setdefault(slot // block, []).append((slot % block, t))
    out = {}
    for name in ("k", "v"):
        value = s[name].double()
        scale = s[name + "_scale"].double()
        x = s[name + "_new"].double().view(-1, kv_heads, hd)
        for b, rows in runs.items():
            first = rows[0][0]
            new = x[[t for _, t in rows]]
            old = scale[b] if first else torch.zeros_like(scale[b])
            now = torch.maximum(old, (new.abs().amax((0, 2)) / top).float().double())
            near = (lambda v: torch.round(v.float()).clamp(-top, top) if kind is torch.int8 else v.float().clamp(-top, top).to(kind))
            if first:
                grown = (value[b, :, :first] * (old / now).float().double()[:, None, None])
                value[b, :, :first] = torch.where((now > old)[:, None, None], near(grown).double(), value[b, :, :first])
            for (o, _), row in zip(rows, new):
                value[b, :, o] = near(row / now[:, None]).double()
            scale[b] = now
        at = s["read"].long()
        out[name] = (value[at // block, :, at % block] * scale[at // block][:, :, None]).reshape(-1, kv_heads * hd)
        out[name + "_scale"] = scale
    return out


def exact_attend(s):
    """Row by row over the row's own positions."""
    c = s["case"]
    block, heads, kv_heads, hd = c["block"], c["heads"], c["kv_heads"], c["head_dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    seqs, spots = s["seq"].tolist(), s["pos"].tolist()
    for r, (z, p) in enumerate(zip(seqs, spots)):
        if p < 0:
            continue
        t = torch.arange(p + 1, device=DEV)
        b = s["table"][z].long()[t // block]
        for h in range(kv_heads):
            k = s["k"][b, h, t % block].double() * s["k_scale"][b, h].double()[:, None]
            v = s["v"][b, h, t % block].double() * s["v_scale"][b, h].double()[:, None]
            q = s["q"][r].double().view(heads, hd)[h::kv_heads]
            out[r].view(heads, hd)[h::kv_heads] = torch.softmax(q @ k.T * s["scale"], 1) @ v
    return out


def exact_prob(s):
    """Each row's draw with weights in 64 bits."""
    c = s["case"]
    got = []
    for r in range(c["rows"]):
        z = s["logits"][r].double()
        t, k, top_p, min_p = (s[n][r].item() for n in ("temperature", "top_k", "top_p", "min_p"))
        if not t > 0:
            got.append(1.0)
            continue
        order = sorted_first(z)
        # the exponent is formed in 32 bits: the operator's inputs are the logits and 1/t as 32-bit numbers
        x = (s["logits"][r].float() - s["logits"][r].float().max()) * (1.0 / s["temperature"][r])
        w = torch.exp(x.double())
        kept = torch.zeros_like(w)
        order = order[:k] if k > 0 else order
        p = w[order]
        if top_p < 1:
            order = order[(p.cumsum(0) - p) < top_p * p.sum()]
        kept[order] = w[order]
        kept = torch.where(w >= min_p, kept, 0.0)
        ends = kept.cumsum(0)
        i = min(int((ends <= s["u"][r].double() * ends[-1]).sum()), c["vocab"] - 1)
        got.append((kept[i] / ends[-1]).item())
    return torch.tensor(got, dtype=torch.float64)


def sorted_first(z):
    """Indices by falling value, equal values by rising index."""
    return torch.sort(-z, stable=True).indices
