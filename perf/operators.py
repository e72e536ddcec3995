"""Measured cases of the paged TurboQuant cache: quantize-on-insert into pages, decode attention over pages (with an
optional sliding window and sink tokens), prompt attention with the same window, reading pages back as dense rows,
and copying pages (forks and compaction).

`run` computes an operator in its plain form (elementary torch operations, 32-bit) while `own` is false, and through
the framework's public entry points while it is true.  `exact` evaluates the definitions in 64 bits.

Vocabulary: a pool holds pages of `page` token positions for every kv head; `page_table[b, i]` is the pool page of
positions [i * page, (i + 1) * page) of sequence b, -1 where the sequence has no page (behind its end, or freed
because it slid out of the window).  Packed rows: code j of a vector sits in word j // per_word at bit
(j % per_word) * bits (3 bits: 10 per word, 4 bits: 8 per word), a vector is
norm * signs * butterfly(centroid[code]) / dim."""

import math
import random

import torch

own = False

DIM = 128
PER_WORD = {3: 10, 4: 8}
# Lloyd-Max centroids of N(0, 1): the codebooks of the packed format
BOOK = {3: [-2.1520, -1.3440, -0.7560, -0.2451, 0.2451, 0.7560, 1.3440, 2.1520],
        4: [-2.7326, -2.0690, -1.6180, -1.2562, -0.9423, -0.6568, -0.3881, -0.1284,
            0.1284, 0.3881, 0.6568, 0.9423, 1.2562, 1.6180, 2.0690, 2.7326]}
DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---- the cases ---------------------------------------------------------------------------------------------------
def listed():
    return [
        # one chat turn of a single user on a 28 / 4 head model, both halves packed: a launch-latency call
        dict(name="decode_one_short", op="decode", batch=1, n_q=28, n_kv=4, min_len=433, max_len=433, page=64,
             kbits=3, vbits=3, dtype="f16", window=0, sinks=0, lens_seed=1),
        # one long document at 32768 tokens, keys kept in 16 bits (the V-only configuration), one sequence only
        dict(name="decode_one_long_dense_k", op="decode", batch=1, n_q=28, n_kv=4, min_len=32768, max_len=32768,
             page=64, kbits=0, vbits=3, dtype="f16", window=0, sinks=0, lens_seed=2),
        # a full serving batch of ragged sequences up to 8192 tokens, K 4-bit + V 3-bit, one empty slot
        dict(name="decode_batch_ragged", op="decode", batch=32, n_q=32, n_kv=8, min_len=700, max_len=8192, page=64,
             kbits=4, vbits=3, dtype="bf16", window=0, sinks=0, lens_seed=3),
        # long chats streamed with a 4096-token window and 4 sink tokens; what slid out has no pages any more
        dict(name="decode_window_stream", op="decode", batch=16, n_q=64, n_kv=8, min_len=20011, max_len=65536, page=128,
             kbits=3, vbits=3, dtype="bf16", window=4096, sinks=4, lens_seed=4),
        # the append of one decode step of a batch (one token per sequence)
        dict(name="append_step", op="append", batch=32, n_kv=8, tokens=1, min_len=700, max_len=8192, page=64,
             kbits=4, vbits=3, dtype="bf16", lens_seed=5),
        # prompts of different lengths inserted together, padded to the longest
        dict(name="append_prompts", op="append", batch=6, n_kv=8, tokens=5000, min_len=0, max_len=3000, page=64,
             kbits=3, vbits=3, dtype="f16", lens_seed=6),
        # one short cached prefix read back for a follow-up prompt
        dict(name="read_prefix_short", op="read", batch=1, n_kv=4, min_len=777, max_len=777, page=64, bits=3,
             dtype="f16", lens_seed=7),
        # shared system prompts of a batch read back before the users' own prompts are attended
        dict(name="read_prefix_batch", op="read", batch=8, n_kv=8, min_len=3001, max_len=16384, page=128, bits=4,
             dtype="bf16", lens_seed=8),
        # a short prompt under a small window: odd length, the tiles at the window's edge dominate
        dict(name="prompt_window_short", op="prompt", batch=1, n_q=28, n_kv=4, seq_q=1001, past=0, window=256, sinks=4,
             dtype="f16"),
        # a long chunk of a prompt behind a cached prefix
        dict(name="prompt_window_chunk", op="prompt", batch=1, n_q=28, n_kv=4, seq_q=7000, past=1192, window=2048,
             sinks=64, dtype="bf16"),
        # forking three sequences: their half-filled last pages are copied in every layer
        dict(name="copy_fork", op="copy", layers=8, n_kv=4, pages=96, copies=3, page=64, kbits=3, vbits=3),
        # compaction of a fragmented pool
        dict(name="copy_compact", op="copy", layers=2, n_kv=8, pages=4500, copies=1500, page=64, kbits=4, vbits=3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "decode", "append", "read", "prompt", "copy"])
    heads = rng.choice([(28, 4), (32, 8), (64, 8), (16, 16), (32, 4), (12, 2)])
    page = rng.choice([32, 64, 128, 256])
    bits = rng.choice([3, 4]), rng.choice([3, 4])
    dtype = rng.choice(["f16", "bf16"])
    seed = rng.randrange(1 << 20)
    if op == "decode":
        batch = _log(rng, 1, 32)
        kbits = rng.choice([0, bits[0], bits[0]])
        longest = _log(rng, 40, min(65536, (1000000 if kbits else 400000) // (batch * heads[1])))
        windowed = rng.random() < 0.4
        return dict(op=op, batch=batch, n_q=heads[0], n_kv=heads[1], min_len=max(1, longest // rng.choice([1, 3, 20])),
                    max_len=longest, page=page, kbits=kbits, vbits=bits[1], dtype=dtype,
                    window=_log(rng, 16, 4096) if windowed else 0, sinks=rng.choice([0, 1, 4, 77]) if windowed else 0,
                    lens_seed=seed)
    if op == "append":
        batch = _log(rng, 1, 32)
        tokens = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, min(5000, 200000 // (batch * heads[1]))))
        return dict(op=op, batch=batch, n_kv=heads[1], tokens=tokens, min_len=0, max_len=_log(rng, 1, 4000), page=page,
                    kbits=rng.choice([0, bits[0], bits[0]]), vbits=bits[1], dtype=dtype, lens_seed=seed)
    if op == "read":
        batch = _log(rng, 1, 8)
        longest = _log(rng, 20, min(16384, 900000 // (batch * heads[1])))
        return dict(op=op, batch=batch, n_kv=heads[1], min_len=max(1, longest // rng.choice([1, 5])), max_len=longest,
                    page=page, bits=bits[0], dtype=dtype, lens_seed=seed)
    if op == "prompt":
        seq = _log(rng, 33, 150000 // heads[0] if heads[0] > 28 else 5000)
        return dict(op=op, batch=rng.choice([1, 1, 2]) if seq < 1500 else 1, n_q=heads[0], n_kv=heads[1], seq_q=seq,
                    past=rng.choice([0, 0, _log(rng, 1, 1500)]), window=_log(rng, 16, 2048), sinks=rng.choice([0, 1, 4, 64, 130]),
                    dtype=dtype)
    layers = rng.choice([1, 2, 5])
    pages = _log(rng, 16, max(20, min(4000, 4000000 // (layers * heads[1] * page))))
    return dict(op=op, layers=layers, n_kv=heads[1], pages=pages, copies=max(1, _log(rng, 1, pages // 2)),
                page=page, kbits=bits[0], vbits=bits[1])


def _lens(case):
    """Token counts of the batch before the call: the longest first, the others spread over the range; a batch of
    eight or more keeps one empty slot, as a serving loop does."""
    r = random.Random(case["lens_seed"])
    lo, hi, n = case["min_len"], case["max_len"], case["batch"]
    got = [hi] + [r.randint(lo, hi) for _ in range(n - 1)]
    if n >= 8 and case["op"] == "decode":
        got[-1] = 0
    return got


def _counts(case):
    """New tokens per sequence of an append: the padded length for the first, fewer for the others."""
    r = random.Random(case["lens_seed"] + 1)
    t = case["tokens"]
    return [t] + [t if t == 1 else r.randint(max(1, t // 3), t) for _ in range(case["batch"] - 1)]


def _words(bits):
    return -(-DIM // PER_WORD[bits])


def _visible(n, window, sinks):
    """How many of n positions the newest one sees."""
    return n if not window else min(n, window) + min(sinks, max(0, n - window))


def work(case):
    op = case["op"]
    if op == "decode":
        row = (2 * DIM if not case["kbits"] else 4 * _words(case["kbits"]) + 4) + 4 * _words(case["vbits"]) + 4
        seen = sum(_visible(n, case["window"], case["sinks"]) for n in _lens(case))
        qo = 2 * case["batch"] * case["n_q"] * DIM * 2
        return {"bytes": seen * case["n_kv"] * row + qo, "flops": 4.0 * seen * case["n_q"] * DIM}
    if op == "append":
        rows = sum(_counts(case)) * case["n_kv"]
        k_out = 2 * DIM if not case["kbits"] else 4 * _words(case["kbits"]) + 4
        return {"bytes": rows * (2 * 2 * DIM + k_out + 4 * _words(case["vbits"]) + 4),
                "flops": rows * DIM * (7 + 4) * (1 if not case["kbits"] else 2)}
    if op == "read":
        rows = sum(_lens(case)) * case["n_kv"]
        out = case["batch"] * max(_lens(case)) * case["n_kv"] * 2 * DIM
        return {"bytes": rows * (4 * _words(case["bits"]) + 4) + out, "flops": rows * DIM * (7 + 2)}
    if op == "prompt":
        n, past = case["seq_q"], case["past"]
        pairs = sum(_visible(past + i + 1, case["window"], case["sinks"]) for i in range(n))
        nbytes = 2 * DIM * case["batch"] * (2 * case["n_q"] * n + 2 * case["n_kv"] * (n + past))
        return {"bytes": nbytes, "flops": 4.0 * DIM * pairs * case["n_q"] * case["batch"]}
    per_page = case["n_kv"] * case["page"] * (4 * _words(case["kbits"]) + 4 * _words(case["vbits"]) + 8)
    return {"bytes": 2 * case["layers"] * case["copies"] * per_page, "flops": 0}


# ---- inputs ------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pack(codes, bits):
    per, n = PER_WORD[bits], _words(bits)
    codes = torch.nn.functional.pad(codes, (0, n * per - DIM)).view(*codes.shape[:-1], n, per)
    shifts = torch.arange(per, device="cuda", dtype=torch.int32) * bits
    return (codes.to(torch.int32) << shifts).sum(-1, dtype=torch.int32)


def _packed_pool(g, pages, n_kv, page, bits):
    """Codes of Gaussian coordinates, as rotated unit vectors have them, and log-normal norms."""
    packed = torch.empty((pages, n_kv, page, _words(bits)), dtype=torch.int32, device="cuda")
    book = torch.tensor(BOOK[bits], device="cuda")
    edges = (book[1:] + book[:-1]) / 2
    for at in range(0, pages, 256):
        n = min(256, pages - at)
        x = torch.randn((n, n_kv, page, DIM), generator=g, device="cuda")
        packed[at:at + n] = _pack(torch.bucketize(x, edges, out_int32=True), bits)
    norms = 11.3 * torch.exp(0.3 * torch.randn((pages, n_kv, page), generator=g, device="cuda"))
    return packed.view(torch.uint32), norms


def _signs(g):
    return torch.randint(0, 2, (DIM,), generator=g, device="cuda").float() * 2 - 1


def _half(g, bits):
    """Codebook, borders and signs of one half (K or V) of a packed cache."""
    book = torch.tensor(BOOK[bits], device="cuda")
    return dict(centroids=book, boundaries=(book[1:] + book[:-1]) / 2, signs=_signs(g), bits=bits)


def _table(g, lens, page, pool, window=0, sinks=0):
    """Shuffled pages of the pool for each sequence, -1 where a sequence holds none."""
    width = max(1, max(-(-n // page) for n in lens))
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    order, at = torch.randperm(pool, generator=torch.Generator().manual_seed(int(torch.randint(1 << 30, (1,), generator=g, device="cuda")))), 0
    for b, n in enumerate(lens):
        for i in range(-(-n // page)):
            if window and i * page >= sinks and (i + 1) * page <= n - window:
                continue
            table[b, i] = order[at]
            at += 1
    return table.cuda(), at


def _pages_needed(lens, page, window=0, sinks=0):
    return sum(1 for n in lens for i in range(-(-n // page))
               if not (window and i * page >= sinks and (i + 1) * page <= n - window))


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = dict(case=case, op=op)
    dtype = DTYPE.get(case.get("dtype"))
    if op in ("decode", "append", "read"):
        lens, page = _lens(case), case["page"]
        window, sinks = case.get("window", 0), case.get("sinks", 0)
        total = [a + b for a, b in zip(lens, _counts(case))] if op == "append" else lens
        pool = _pages_needed(total, page, window, sinks) + 3
        s["table"], _ = _table(g, total, page, pool, window, sinks)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        n_kv = case["n_kv"]
        vbits = case["bits"] if op == "read" else case["vbits"]
        v = dict(format="polar", **_half(g, vbits))
        v["packed"], v["norms"] = _packed_pool(g, pool, n_kv, page, vbits)
        s["v"] = v
        if op != "read":
            if case["kbits"]:
                k = dict(format="polar", **_half(g, case["kbits"]))
                k["packed"], k["norms"] = _packed_pool(g, pool, n_kv, page, case["kbits"])
            else:
                k = dict(format="dense", data=torch.randn((pool, n_kv, page, DIM), generator=g, device="cuda").to(dtype))
            s["k"] = k
        if op == "decode":
            s["q"] = torch.randn((case["batch"], case["n_q"], DIM), generator=g, device="cuda").to(dtype)
        if op == "append":
            shape = (case["batch"], case["tokens"], n_kv, DIM)        # projections come out token-major
            s["keys"] = torch.randn(shape, generator=g, device="cuda").to(dtype).transpose(1, 2)
            vals = torch.randn(shape, generator=g, device="cuda") * torch.exp(
                0.5 * torch.randn(shape[:3], generator=g, device="cuda"))[..., None]
            s["values"] = vals.to(dtype).transpose(1, 2)
            s["counts"] = torch.tensor(_counts(case), dtype=torch.int32, device="cuda")
        if op == "read":
            s["length"] = max(lens)
            s["dtype"] = dtype
    elif op == "prompt":
        n, total = case["seq_q"], case["seq_q"] + case["past"]
        mk = lambda h, m: torch.randn((case["batch"], m, h, DIM), generator=g, device="cuda").to(dtype).transpose(1, 2)  # noqa: E731
        s["q"], s["k"], s["v"] = mk(case["n_q"], n), mk(case["n_kv"], total), mk(case["n_kv"], total)
    else:
        s["pools"] = []
        for _ in range(case["layers"]):
            for bits in (case["kbits"], case["vbits"]):
                shape = (case["pages"], case["n_kv"], case["page"])
                s["pools"].append(torch.randint(0, 1 << 30, shape + (_words(bits),), generator=g, device="cuda",
                                                dtype=torch.int32).view(torch.uint32))
                s["pools"].append(torch.rand(shape, generator=g, device="cuda") * 9 + 1)
        order = torch.randperm(case["pages"], generator=g, device="cuda").to(torch.int32)
        s["src"], s["dst"] = order[:case["copies"]].clone(), order[case["copies"]:2 * case["copies"]].clone()
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------
def _butterfly(x):
    """Raw Walsh-Hadamard butterfly of the last dimension: stages 1, 2, 4, ... of (a + b, a - b)."""
    shape, h = x.shape, 1
    while h < DIM:
        x = x.reshape(*shape[:-1], DIM // (2 * h), 2, h)
        x = torch.stack((x[..., 0, :] + x[..., 1, :], x[..., 0, :] - x[..., 1, :]), dim=-2)
        h *= 2
    return x.reshape(shape)


def _unpack(words, bits):
    shifts = torch.arange(PER_WORD[bits], device=words.device, dtype=torch.int32) * bits
    codes = (words.view(torch.int32).unsqueeze(-1) >> shifts) & ((1 << bits) - 1)
    return codes.flatten(-2)[..., :DIM]


def _gather(pool, table):
    """(pages, heads, page, ...) by table (B, width) -> (B, heads, width * page, ...); absent pages read page 0."""
    got = pool[table.clamp(min=0).long()].transpose(1, 2)
    return got.flatten(2, 3)


def _plain_decode(s):
    c, k, v, q = s["case"], s["k"], s["v"], s["q"].float()
    n_kv, rep = c["n_kv"], c["n_q"] // c["n_kv"]
    q = q.view(c["batch"], n_kv, rep, DIM)
    if k["format"] == "polar":
        q = _butterfly(q * k["signs"])
        rows = k["centroids"][_unpack(_gather(k["packed"].view(torch.int32), s["table"]), k["bits"])]
        scores = (q @ rows.transpose(-1, -2)) * (_gather(k["norms"], s["table"]) / DIM)[:, :, None]
    else:
        scores = q @ _gather(k["data"], s["table"]).float().transpose(-1, -2)
    scores = scores * DIM ** -0.5
    at = torch.arange(scores.shape[-1], device=q.device)
    n = s["lens"].long()[:, None]
    seen = at < n
    if c["window"]:
        seen = seen & ((at >= n - c["window"]) | (at < c["sinks"]))
    scores = torch.where(seen[:, None, None], scores, float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    rows = v["centroids"][_unpack(_gather(v["packed"].view(torch.int32), s["table"]), v["bits"])]
    out = (p * torch.where(seen[:, None], _gather(v["norms"], s["table"]), 0.0)[:, :, None]) @ rows
    out = v["signs"] * _butterfly(out) / DIM
    out = torch.where(total > 0, out / total, 0.0)
    return out.reshape(c["batch"], c["n_q"], DIM).to(s["q"].dtype)


def _plain_codes(x, half):
    """Words and norms of rows x: the format defines its codes by these 32-bit steps in this order, so that every
    implementation gets the same words."""
    x = x.float()
    ss = x * x
    while ss.shape[-1] > 1:
        ss = ss[..., 0::2] + ss[..., 1::2]
    norm = ss.sqrt()
    raw = _butterfly(x / norm.clamp(min=1e-8) * half["signs"])
    scale = torch.full((), 1.0 / math.sqrt(DIM), dtype=torch.float32, device=x.device)
    codes = torch.bucketize(raw * scale / scale, half["boundaries"], out_int32=True)
    return _pack(codes, half["bits"]), norm[..., 0]


def _places(s):
    c = s["case"]
    step = torch.arange(c["tokens"], device="cuda")
    pos = s["lens"].long()[:, None] + step
    live = step < s["counts"].long()[:, None]
    b, t = live.nonzero(as_tuple=True)
    pos = pos[b, t]
    return b, t, s["table"].long()[b, pos // c["page"]], pos % c["page"]


def _plain_append(s):
    b, t, page, row = _places(s)
    for x, half in ((s["keys"], s["k"]), (s["values"], s["v"])):
        x = x.transpose(1, 2)[b, t]
        if half["format"] == "dense":
            half["data"][page, :, row] = x
        else:
            words, norms = _plain_codes(x, half)
            half["packed"].view(torch.int32)[page, :, row] = words
            half["norms"][page, :, row] = norms
    return _appended(s)


def _appended(s):
    k, v = s["k"], s["v"]
    keys = [k["data"]] if k["format"] == "dense" else [k["packed"].view(torch.int32), k["norms"]]
    return keys + [v["packed"].view(torch.int32), v["norms"]]


def _plain_read(s):
    v, n = s["v"], s["length"]
    width = -(-n // s["case"]["page"])
    table = s["table"][:, :width]
    scale = torch.full((), 1.0 / math.sqrt(DIM), dtype=torch.float32, device="cuda")
    rows = v["centroids"][_unpack(_gather(v["packed"].view(torch.int32), table)[:, :, :n], v["bits"])] * scale
    rows = _butterfly(rows) * scale * v["signs"] * _gather(v["norms"], table)[:, :, :n, None]
    live = torch.arange(n, device="cuda") < s["lens"].long()[:, None]
    return torch.where(live[:, None, :, None], rows, 0.0).to(s["dtype"])


def _plain_prompt(s):
    c, q, k, v = s["case"], s["q"].float(), s["k"].float(), s["v"].float()
    rep = c["n_q"] // c["n_kv"]
    scores = q.unflatten(1, (c["n_kv"], rep)) @ k[:, :, None].transpose(-1, -2)
    i = torch.arange(c["seq_q"], device="cuda")[:, None] + c["past"]
    j = torch.arange(c["seq_q"] + c["past"], device="cuda")
    seen = (j <= i) & ((j > i - c["window"]) | (j < c["sinks"]))
    scores.mul_(DIM ** -0.5).masked_fill_(~seen, float("-inf"))
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    return ((scores @ v[:, :, None]) / total).flatten(1, 2).to(s["q"].dtype)


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    for pool in s["pools"]:
        pool = pool.view(torch.int32) if pool.dtype == torch.uint32 else pool
        pool[dst] = pool[src]
    return _copied(s)


def _copied(s):
    return [p.view(torch.int32) if p.dtype == torch.uint32 else p for p in s["pools"]]


PLAIN = dict(decode=_plain_decode, append=_plain_append, read=_plain_read, prompt=_plain_prompt, copy=_plain_copy)


# ---- the framework's calls -----------------------------------------------------------------------------------------
def _package():
    import __graft_entry__
    return __graft_entry__.load_package()


def _own_decode(s):
    c = s["case"]
    return _package().paged_decode(s["q"], k=s["k"], v=s["v"], page_table=s["table"], seq_lens=s["lens"],
                                   attn_scale=DIM ** -0.5, window=c["window"], sinks=c["sinks"])


def _own_append(s):
    _package().paged_append(s["keys"], s["values"], k=s["k"], v=s["v"], page_table=s["table"], starts=s["lens"],
                            counts=s["counts"])
    return _appended(s)


def _own_read(s):
    return _package().paged_dequantize(s["v"], page_table=s["table"], seq_lens=s["lens"], length=s["length"],
                                       dtype=s["dtype"])


def _own_prompt(s):
    c = s["case"]
    return _package().prefill_attention(s["q"], s["k"], s["v"], DIM ** -0.5, causal=True, window=c["window"],
                                        sinks=c["sinks"])


def _own_copy(s):
    _package().copy_pages(s["pools"], s["src"], s["dst"])
    return _copied(s)


OWN = dict(decode=_own_decode, append=_own_append, read=_own_read, prompt=_own_prompt, copy=_own_copy)


def run(state):
    return (OWN if own else PLAIN)[state["op"]](state)


# ---- 64-bit values ---------------------------------------------------------------------------------------------------
def _hadamard64():
    h = torch.ones((1, 1), dtype=torch.float64, device="cuda")
    while h.shape[0] < DIM:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)))
    return h


def _rows64(half, b_table, n, page):
    """Positions [0, n) of one sequence in 64 bits: (heads, n, dim)."""
    pages = b_table[:-(-n // page)].clamp(min=0).long()
    words = half["packed"].view(torch.int32)[pages].to(torch.int64)
    codes = [(words[..., j // PER_WORD[half["bits"]]] >> (j % PER_WORD[half["bits"]] * half["bits"])) % (1 << half["bits"])
             for j in range(DIM)]
    book = torch.tensor(BOOK[half["bits"]], dtype=torch.float32, device="cuda").double()
    rows = book[torch.stack(codes, -1)] @ _hadamard64() * half["signs"].double() / DIM
    rows = rows * half["norms"][pages].double().unsqueeze(-1)
    return rows.permute(1, 0, 2, 3).reshape(rows.shape[1], -1, DIM)[:, :n]


def _exact_decode(s):
    c, k, v = s["case"], s["k"], s["v"]
    out = torch.zeros((c["batch"], c["n_q"], DIM), dtype=torch.float64, device="cuda")
    rep = c["n_q"] // c["n_kv"]
    for b, n in enumerate(_lens(c)):
        if n == 0:
            continue
        if k["format"] == "polar":
            keys = _rows64(k, s["table"][b], n, c["page"])
        else:
            pages = s["table"][b, :-(-n // c["page"])].clamp(min=0).long()
            keys = k["data"][pages].double().permute(1, 0, 2, 3).reshape(c["n_kv"], -1, DIM)[:, :n]
        vals = _rows64(v, s["table"][b], n, c["page"])
        at = [j for j in range(n) if not c["window"] or j >= n - c["window"] or j < c["sinks"]]
        at = torch.tensor(at, device="cuda")
        keys, vals = keys[:, at], vals[:, at]
        for h in range(c["n_q"]):
            w = torch.softmax(keys[h // rep] @ s["q"][b, h].double() / math.sqrt(DIM), 0)
            out[b, h] = w @ vals[h // rep]
    return out


def _exact_append(s):
    """Norms in 64 bits and the dense rows as they are.  The words have no 64-bit value: the format defines them by
    32-bit steps, and a value next to a border may fall on its other side in 64."""
    c = s["case"]
    out = []
    for x, half in ((s["keys"], s["k"]), (s["values"], s["v"])):
        pool = (half["data"] if half["format"] == "dense" else half["norms"]).double()
        for b, (start, count) in enumerate(zip(_lens(c), _counts(c))):
            pos = torch.arange(start, start + count, device="cuda")
            page = s["table"][b].long()[pos // c["page"]]
            rows = x[b, :, :count].double().transpose(0, 1)
            pool[page, :, pos % c["page"]] = rows if half["format"] == "dense" else torch.linalg.vector_norm(rows, dim=-1)
        out += [pool] if half["format"] == "dense" else [None, pool]
    return out


def _exact_read(s):
    c = s["case"]
    out = torch.zeros((c["batch"], c["n_kv"], s["length"], DIM), dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lens(c)):
        out[b, :, :n] = _rows64(s["v"], s["table"][b], n, c["page"])
    return out


def _exact_prompt(s):
    c = s["case"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    rep, past = c["n_q"] // c["n_kv"], c["past"]
    for b in range(c["batch"]):
        for h in range(c["n_q"]):
            q, k, v = s["q"][b, h].double(), s["k"][b, h // rep].double(), s["v"][b, h // rep].double()
            for at in range(0, c["seq_q"], 2048):
                rows = torch.arange(at, min(at + 2048, c["seq_q"]), device="cuda") + past
                gap = rows[:, None] - torch.arange(k.shape[0], device="cuda")[None]
                hidden = (gap < 0) | ((gap >= c["window"]) & (torch.arange(k.shape[0], device="cuda") >= c["sinks"])[None])
                w = torch.softmax((q[rows - past] @ k.T / math.sqrt(DIM)).masked_fill(hidden, -math.inf), -1)
                out[b, h, rows - past] = w @ v
    return out


def _exact_copy(s):
    """Moved values are as they were; whole words have no other form."""
    out = []
    for pool in s["pools"]:
        if pool.dtype == torch.uint32:
            out.append(None)
        else:
            moved = pool.double()
            moved[s["dst"].long()] = pool.double()[s["src"].long()]
            out.append(moved)
    return out


EXACT = dict(decode=_exact_decode, append=_exact_append, read=_exact_read, prompt=_exact_prompt, copy=_exact_copy)


def exact(case, seed):
    return EXACT[case["op"]](prepare(case, seed))
