"""What is measured of the paged cache's operators and of the prompt attention.

    prompt  pf_prompt_attention: causal attention over packed prompts of different lengths, grouped heads
    store   pf_paged_store: the new tokens' keys and values into the pages of a paged cache
    decode  pf_paged_attention: attention of the newest 1 to 8 tokens of every sequence over the paged cache
    fork    pf_paged_free + pf_paged_fork: sequences given up, and others that take a parent's history over
    compact pf_paged_compact: the pages in use moved to the front of the cache

Each operator has its plain form here, in elementary torch operations in 32
bits, and the definition in 64 bits (`exact`).  The paged cache is laid out
[page][layer][kv head][slot][dim], int8 with one scale per row or bf16 / fp16;
`table[seq]` lists a sequence's pages in order, `lens` its tokens, `refs` the
number of sequences that hold a page.
"""
import ctypes
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i8": torch.int8}
CODES = {"f32": 0, "bf16": 1, "f16": 2, "i8": 3}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "i8": 1}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one short request beside two even shorter ones on a small model: what counts is the latency of one launch
        dict(name="prompt, 3 short", op="prompt", seqs=3, shortest=1, longest=131, heads=8, kv_heads=2, dim=64,
             type="f16", fused=True, lens=1),
        # a batch of prompts as the benchmark's (64 sequences of about 512 tokens, 32 and 8 heads), ragged
        dict(name="prompt, 64 ragged", op="prompt", seqs=64, shortest=33, longest=1024, heads=32, kv_heads=8, dim=64,
             type="bf16", fused=False, lens=2),
        # one long document
        dict(name="prompt, 8192 tokens", op="prompt", seqs=1, shortest=8192, longest=8192, heads=32, kv_heads=8,
             dim=128, type="bf16", fused=True, lens=3),
        # a verify step of the benchmark's batch: 5 new tokens for each of 64 sequences into an int8 cache
        dict(name="store, 64 x 5 rows", op="store", seqs=64, fewest=5, most=5, before=700, kv_heads=8, dim=64,
             page=64, type="f32", cache="i8", layers=1, lens=4),
        # a whole batch of prompts into the cache
        dict(name="store, 64 prompts", op="store", seqs=64, fewest=100, most=1000, before=1, kv_heads=8, dim=64,
             page=64, type="f32", cache="i8", layers=1, lens=5),
        # one user, an ordinary context, one token: latency
        dict(name="decode, 1 x 777", op="decode", seqs=1, rows=1, shortest=777, longest=777, heads=32, kv_heads=8,
             dim=64, page=16, type="f32", cache="i8", layers=2, lens=6),
        # a verify step of the benchmark's batch: 4 drafts and the pending token, contexts of 512 to 1024
        dict(name="decode, 64 x 5 rows", op="decode", seqs=64, rows=5, shortest=512, longest=1024, heads=32,
             kv_heads=8, dim=64, page=64, type="f32", cache="i8", layers=1, lens=7),
        # a few long contexts, the longest 65,536 tokens, beside short ones
        dict(name="decode, long", op="decode", seqs=8, rows=1, shortest=3000, longest=65536, heads=32, kv_heads=8,
             dim=128, page=64, type="bf16", cache="bf16", layers=1, lens=8),
        # two beams of four on a small model
        dict(name="fork, 2 x 4", op="fork", parents=2, fan=4, shortest=90, longest=200, kv_heads=8, dim=64, page=16,
             cache="i8", layers=2, spare=64, lens=9),
        # sixteen prompts with eight continuations each, every layer of the benchmark's model
        dict(name="fork, 16 x 8", op="fork", parents=16, fan=8, shortest=200, longest=2048, kv_heads=8, dim=64,
             page=64, cache="i8", layers=22, spare=32, lens=10),
        # a small cache after a few requests have left
        dict(name="compact, 256 pages", op="compact", seqs=12, shortest=60, longest=400, pages=256, kv_heads=8, dim=64,
             page=16, cache="i8", layers=2, lens=11),
        # a cache of 1,024 pages, about half of them in use, every layer of the benchmark's model
        dict(name="compact, 1024 pages", op="compact", seqs=48, shortest=300, longest=1500, pages=1024, kv_heads=8,
             dim=64, page=64, cache="i8", layers=22, lens=12),
    ]


def spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["prompt", "store", "decode", "fork", "compact"])
    kv = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 128])
    lens = rng.randrange(1 << 30)
    page = rng.choice([16, 32, 64, 128])
    if op == "prompt":
        group = rng.choice([1, 2, 3, 4, 7, 8])
        kv = min(kv, 32 // group)
        longest = spread(rng, 1, 4096)
        seqs = spread(rng, 1, max(1, min(96, 16384 // longest)))
        return dict(op=op, seqs=seqs, shortest=spread(rng, 1, longest), longest=longest, heads=kv * group, kv_heads=kv,
                    dim=dim, type=rng.choice(["bf16", "f16"]), fused=rng.random() < 0.5, lens=lens)
    cache = rng.choice(["i8", "i8", "bf16", "f16"])
    if op == "store":
        most = spread(rng, 1, 1000)
        return dict(op=op, seqs=spread(rng, 1, max(1, min(128, 16384 // most))), fewest=spread(rng, 1, most), most=most,
                    before=spread(rng, 1, 2000), kv_heads=kv, dim=dim, page=page,
                    type=rng.choice(["f32", "bf16", "f16"]) if cache == "i8" else rng.choice(["f32", cache]), cache=cache,
                    layers=rng.choice([1, 2]), lens=lens)
    if op == "decode":
        longest = spread(rng, 8, 32768)
        seqs = spread(rng, 1, max(1, min(128, (1 << 20) // (longest * kv))))
        return dict(op=op, seqs=seqs, rows=rng.choice([1, 1, 1, 2, 3, 5, 8]), shortest=spread(rng, 1, longest),
                    longest=longest, heads=kv * rng.choice([1, 2, 3, 4, 5, 8]), kv_heads=kv, dim=dim, page=page,
                    type=rng.choice(["f32", "bf16", "f16"]) if cache == "i8" else cache, cache=cache, layers=1, lens=lens)
    layers = rng.choice([1, 2, 5, 22])
    if op == "fork":
        longest = spread(rng, 1, 2048)
        return dict(op=op, parents=spread(rng, 1, 12), fan=rng.choice([1, 2, 3, 5, 8]), shortest=spread(rng, 1, longest),
                    longest=longest, kv_heads=kv, dim=64, page=page, cache=cache, layers=layers, spare=rng.randint(1, 40),
                    lens=lens)
    longest = spread(rng, page, 1500)
    seqs = spread(rng, 2, 32)
    return dict(op=op, seqs=seqs, shortest=spread(rng, 1, longest), longest=longest,
                pages=int(seqs * -(-longest // page) * rng.uniform(1.0, 2.5)) + 1, kv_heads=kv, dim=64, page=page,
                cache=cache, layers=layers, lens=lens)


def lengths(c, n, low, high):
    """n lengths between low and high, both among them, from the case alone."""
    rng = random.Random(c["lens"])
    got = [high, low][:n] + [spread(rng, low, high) for _ in range(n - 2)]
    rng.shuffle(got)
    return got


# ---------------------------------------------------------------------------
# States
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    s = dict(case)
    {"prompt": prepare_prompt, "store": prepare_store, "decode": prepare_decode, "fork": prepare_fork,
     "compact": prepare_compact}[case["op"]](case, s, g)
    return s


def normal(g, shape, t, by=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32 if t == torch.float32 else torch.float16)
            * by).to(t)


def prepare_prompt(c, s, g):
    """Queries, keys and values of packed prompts; `fused`: columns of one buffer, as a joined projection leaves them."""
    n = lengths(c, c["seqs"], c["shortest"], c["longest"])
    offsets = [0]
    for x in n:
        offsets.append(offsets[-1] + x)
    t, d = TYPES[c["type"]], c["dim"]
    cols = [c["heads"] * d, c["kv_heads"] * d, c["kv_heads"] * d]
    if c["fused"]:
        rows = normal(g, (offsets[-1], sum(cols)), t)
        s["q"], s["k"], s["v"] = rows.split(cols, dim=1)
    else:
        s["q"], s["k"], s["v"] = (normal(g, (offsets[-1], w), t) for w in cols)
    s["out"] = torch.empty(offsets[-1], cols[0], dtype=t, device="cuda")
    s["n_tokens"], s["offsets"] = offsets[-1], torch.tensor(offsets, dtype=torch.int32, device="cuda")
    s["scale"] = 1 / math.sqrt(d)


def cache_of(c, s, g, n_pages, used, max_pages, at_random=True):
    """A cache of n_pages pages; `used`: for each sequence its tokens.  Pages in an order as after some time of use."""
    rng = random.Random(c["lens"] + 1)
    order = rng.sample(range(n_pages), n_pages) if at_random else list(range(n_pages))
    t, shape = TYPES[c["cache"]], (n_pages, c["layers"], c["kv_heads"], c["page"])
    s["ks"] = s["vs"] = None
    if c["cache"] == "i8":
        s["k"], s["v"] = (torch.randint(-127, 128, (*shape, c["dim"]), generator=g, device="cuda", dtype=torch.int8)
                          for _ in range(2))
        s["ks"], s["vs"] = (torch.rand(shape, generator=g, device="cuda") * 0.01 + 0.01 for _ in range(2))
    else:
        s["k"], s["v"] = (normal(g, (*shape, c["dim"]), t) for _ in range(2))
    table, at = [], 0
    for n in used:
        p = -(-n // c["page"])
        table.append(order[at:at + p] + [-1] * (max_pages - p))
        at += p
    refs = [0] * n_pages
    for p in order[:at]:
        refs[p] = 1
    s["n_pages"], s["max_pages"], s["max_seqs"] = n_pages, max_pages, len(used)
    s["table"] = torch.tensor(table, dtype=torch.int32, device="cuda")
    s["lens_now"] = torch.tensor(used, dtype=torch.int32, device="cuda")
    s["refs"] = torch.tensor(refs, dtype=torch.int32, device="cuda")
    return order[at:]


def pages_of(c, n):
    return sum(-(-x // c["page"]) for x in n)


def prepare_store(c, s, g):
    """`lens_now` counts the new tokens already, as after pf_paged_reserve."""
    new = lengths(c, c["seqs"], c["fewest"], c["most"])
    used = [c["before"] + x for x in new]
    cache_of(c, s, g, pages_of(c, used) + 3, used, -(-max(used) // c["page"]))
    offsets = [0]
    for x in new:
        offsets.append(offsets[-1] + x)
    shape = (offsets[-1], c["kv_heads"] * c["dim"])
    s["new_k"], s["new_v"] = (normal(g, shape, TYPES[c["type"]]) for _ in range(2))
    s["n_tokens"], s["offsets"] = offsets[-1], torch.tensor(offsets, dtype=torch.int32, device="cuda")


def prepare_decode(c, s, g):
    used = lengths(c, c["seqs"], c["shortest"], c["longest"])
    cache_of(c, s, g, pages_of(c, used) + 3, used, -(-max(used) // c["page"]))
    shape = (c["seqs"] * c["rows"], c["heads"] * c["dim"])
    s["q"] = normal(g, shape, TYPES[c["type"]], 1.5)
    s["out"] = torch.empty(shape, dtype=TYPES[c["type"]], device="cuda")
    s["scale"] = 1 / math.sqrt(c["dim"])


def fork_lens(c):
    return lengths(c, c["parents"], c["shortest"], c["longest"])


def prepare_fork(c, s, g):
    """Parents with their pages; each child takes a whole history over.  From the second pass on the children still
    hold what the pass before gave them, as the beams of a search do."""
    n = fork_lens(c)
    kids = c["parents"] * c["fan"]
    cache_of(c, s, g, pages_of(c, n) + kids + c["spare"], n + [0] * kids, -(-max(n) // c["page"]) + 1)
    s["parents_at"] = torch.arange(c["parents"], dtype=torch.int32, device="cuda").repeat_interleave(c["fan"])
    s["children_at"] = torch.arange(c["parents"], c["parents"] + kids, dtype=torch.int32, device="cuda")


def compact_layout(c):
    """(lens, table rows, refs) of a fragmented cache: every third sequence shares the full pages of the one before."""
    n = lengths(c, c["seqs"], c["shortest"], c["longest"])
    rng = random.Random(c["lens"] + 1)
    order = rng.sample(range(c["pages"]), c["pages"])
    most = -(-max(n) // c["page"])
    table, refs, at = [], [0] * c["pages"], 0
    for i, x in enumerate(n):
        need = -(-x // c["page"])
        shared = table[-1][:min(n[i - 1], x) // c["page"]] if i % 3 == 2 else []
        own_pages = order[at:at + need - len(shared)]
        at += len(own_pages)
        row = shared + own_pages
        for p in row:
            refs[p] += 1
        table.append(row + [-1] * (most - need))
    return n, table, refs


def prepare_compact(c, s, g):
    n, table, refs = compact_layout(c)
    cache_of(c, s, g, c["pages"], [0] * len(n), len(table[0]))
    s["lens_now"] = torch.tensor(n, dtype=torch.int32, device="cuda")
    s["table_then"] = torch.tensor(table, dtype=torch.int32, device="cuda")
    s["refs_then"] = torch.tensor(refs, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    op = state["op"]
    if own:
        return {"prompt": own_prompt, "store": own_store, "decode": own_decode, "fork": own_fork,
                "compact": own_compact}[op](state)
    return {"prompt": plain_prompt, "store": plain_store, "decode": plain_decode, "fork": plain_fork,
            "compact": plain_compact}[op](state)


def pages_out(s):
    """The cache's pages.  The int8 codes are whole numbers and have to be equal; what they stand for is code x scale."""
    return [s["k"], s["v"]] + ([s["ks"], s["vs"]] if s["ks"] is not None else [])


# ---- the framework's calls ----
def library():
    from pocketforge_b200 import _lib
    return _lib


def own_cache(s):
    """The cache's description, made once for a state as a program does once for its cache."""
    if "cache_c" not in s:
        lib = library()
        c = lib.PagedCacheC(dtype=CODES[s["cache"]], n_layers=s["layers"], n_kv_heads=s["kv_heads"], head_dim=s["dim"],
                            page_size=s["page"], n_pages=s["n_pages"], max_seqs=s["max_seqs"],
                            max_pages=s["max_pages"], k=s["k"].data_ptr(), v=s["v"].data_ptr(),
                            k_scale=s["ks"].data_ptr() if s["ks"] is not None else None,
                            v_scale=s["vs"].data_ptr() if s["vs"] is not None else None,
                            table=s["table"].data_ptr(), lens=s["lens_now"].data_ptr(), refs=s["refs"].data_ptr())
        s["page_work"] = torch.zeros(lib.lib().pf_paged_work_bytes(ctypes.byref(c)), dtype=torch.uint8, device="cuda")
        c.work = s["page_work"].data_ptr()
        s["cache_c"], s["cache_ref"] = c, ctypes.byref(c)
    return s["cache_ref"]


def own_prompt(s):
    lib, q, k, v, out = library(), s["q"], s["k"], s["v"], s["out"]
    lib.check(lib.lib().pf_prompt_attention(
        q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), out.data_ptr(), out.stride(0),
        CODES[s["type"]], s["offsets"].data_ptr(), s["seqs"], s["n_tokens"], s["heads"], s["kv_heads"], s["dim"],
        s["scale"], torch.cuda.current_stream().cuda_stream), "pf_prompt_attention")
    return out


def own_store(s):
    lib, k, v = library(), s["new_k"], s["new_v"]
    lib.check(lib.lib().pf_paged_store(
        own_cache(s), s["layers"] - 1, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), CODES[s["type"]],
        s["offsets"].data_ptr(), s["seqs"], s["n_tokens"], torch.cuda.current_stream().cuda_stream), "pf_paged_store")
    return pages_out(s)


def own_decode(s):
    lib, cache, q, out = library(), own_cache(s), s["q"], s["out"]
    if "work" not in s:
        n = lib.lib().pf_paged_attention_work_bytes(cache, s["seqs"], s["rows"], s["heads"])
        s["work"] = torch.zeros(n, dtype=torch.uint8, device="cuda")
    lib.check(lib.lib().pf_paged_attention(
        cache, s["layers"] - 1, q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), CODES[s["type"]], s["seqs"],
        s["rows"], s["heads"], s["scale"], s["work"].data_ptr(), s["work"].numel(),
        torch.cuda.current_stream().cuda_stream), "pf_paged_attention")
    return out


def own_fork(s):
    lib, cache, st = library(), own_cache(s), torch.cuda.current_stream().cuda_stream
    n = s["children_at"].numel()
    lib.check(lib.lib().pf_paged_free(cache, s["children_at"].data_ptr(), n, st), "pf_paged_free")
    lib.check(lib.lib().pf_paged_fork(cache, s["parents_at"].data_ptr(), s["children_at"].data_ptr(), n, st),
              "pf_paged_fork")
    return pages_out(s) + [s["table"], s["refs"], s["lens_now"]]


def own_compact(s):
    """A pass begins with the fragmented tables, which the pass before has put in order."""
    lib, cache = library(), own_cache(s)
    s["table"].copy_(s["table_then"])
    s["refs"].copy_(s["refs_then"])
    lib.check(lib.lib().pf_paged_compact(cache, torch.cuda.current_stream().cuda_stream), "pf_paged_compact")
    return pages_out(s) + [s["table"], s["refs"]]


# ---- the plain forms ----
def softmax_rows(x):
    """Softmax over the last axis; a row without an entry gives zeros."""
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    n = p.sum(-1, keepdim=True)
    return p / torch.where(n == 0, 1.0, n)


def plain_prompt(s):
    """Padded to the longest prompt: scores, causal mask, softmax, weighted sum."""
    off, d, longest = s["offsets"].long(), s["dim"], s["longest"]
    n = off[1:] - off[:-1]
    pos = torch.arange(longest, device="cuda")
    real = pos < n[:, None]                                               # [seq][pos]
    at = torch.where(real, off[:-1, None] + pos, 0)
    group = s["heads"] // s["kv_heads"]
    q = s["q"][at].float().view(s["seqs"], longest, s["kv_heads"], group, d)
    k, v = (s[x][at].float().view(s["seqs"], longest, s["kv_heads"], d) for x in ("k", "v"))
    v = torch.where(real[:, :, None, None], v, 0.0)
    x = torch.matmul(q.permute(0, 2, 3, 1, 4), k.permute(0, 2, 3, 1)[:, :, None]) * s["scale"]  # [seq][kv][g][q][k]
    x.masked_fill_(pos > pos[:, None], -math.inf)
    o = torch.matmul(softmax_rows(x), v.permute(0, 2, 1, 3)[:, :, None])  # [seq][kv][g][q][d]
    s["out"][at[real]] = o.permute(0, 3, 1, 2, 4).reshape(s["seqs"], longest, -1)[real].to(s["out"].dtype)
    return s["out"]


def row_codes(x):
    """(codes, scale) of rows of values: scale = largest / 127, codes = value * (127 / largest), halves away from zero.
    Each quotient is rounded once: a Python number as an operand would make it a product with a rounded reciprocal."""
    big = x.abs().amax(-1)
    one, most = big == 0, torch.full_like(big, 127.0)
    y = x * torch.where(one, 1.0, most / torch.where(one, 1.0, big))[..., None]
    low = y.abs().floor()
    code = torch.where(y.abs() - low >= 0.5, low + 1, low) * y.sign()
    return code.to(torch.int8), torch.where(one, 1.0, big / most)


def slots_of(s):
    """(page, slot) of every new token: the last ones of each sequence."""
    off = s["offsets"].long()
    i = torch.arange(s["n_tokens"], device="cuda")
    seq = torch.searchsorted(off, i, right=True) - 1
    pos = s["lens_now"][seq] - (off[seq + 1] - i)
    return s["table"][seq, pos // s["page"]].long(), pos % s["page"]


def plain_store(s):
    page, slot = slots_of(s)
    shape, layer = (s["n_tokens"], s["kv_heads"], s["dim"]), s["layers"] - 1
    k, v = s["new_k"].view(shape).float(), s["new_v"].view(shape).float()
    if s["cache"] == "i8":
        k, scale = row_codes(k)
        s["ks"][page, layer, :, slot] = scale
        v, scale = row_codes(v)
        s["vs"][page, layer, :, slot] = scale
    s["k"][page, layer, :, slot] = k.to(s["k"].dtype)
    s["v"][page, layer, :, slot] = v.to(s["v"].dtype)
    return pages_out(s)


def history(s, what, scale, t):
    """[seq][kv head][position][dim] of the whole table's width, in type t."""
    pages = s["table"].clamp(min=0).long()
    x = s[what][pages, s["layers"] - 1].to(t)
    if s["ks"] is not None:
        x *= s[scale][pages, s["layers"] - 1].to(t)[..., None]
    return x.transpose(1, 2).reshape(s["seqs"], s["kv_heads"], -1, s["dim"])


def plain_decode(s):
    b, r, kv, d = s["seqs"], s["rows"], s["kv_heads"], s["dim"]
    group = s["heads"] // kv
    k, v = history(s, "k", "ks", torch.float32), history(s, "v", "vs", torch.float32)
    pos = torch.arange(k.shape[2], device="cuda")
    v = torch.where((pos < s["lens_now"][:, None])[:, None, :, None], v, 0.0)
    q = s["q"].float().view(b, r, kv, group, d).permute(0, 2, 1, 3, 4).reshape(b, kv, r * group, d)
    x = (torch.matmul(q, k.transpose(2, 3)) * s["scale"]).view(b, kv, r, group, -1)
    last = s["lens_now"][:, None] - r + 1 + torch.arange(r, device="cuda")     # entries that row t sees
    x.masked_fill_((pos >= last[..., None])[:, None, :, None], -math.inf)
    o = torch.matmul(softmax_rows(x).view(b, kv, r * group, -1), v).view(b, kv, r, group, d)
    s["out"].copy_(o.permute(0, 2, 1, 3, 4).reshape(b * r, -1))
    return s["out"]


def plain_fork(s):
    """Frees the children, shares the parents' full pages, and copies what the parents hold of a last, partly filled
    page into the lowest free pages."""
    kids, par, size = s["children_at"].long(), s["parents_at"].long(), s["page"]
    held = s["table"][kids]
    s["refs"].index_add_(0, held.clamp(min=0).view(-1).long(), -(held.view(-1) >= 0).int())
    n = s["lens_now"][par].long()
    row = s["table"][par]
    tail, slot = n // size, n % size
    cut = torch.arange(s["max_pages"], device="cuda") < tail[:, None]
    free = (s["refs"] == 0).nonzero().view(-1)
    some = slot > 0
    fresh = free[:int(some.sum())]
    old = row.gather(1, tail.clamp(max=s["max_pages"] - 1)[:, None])[:, 0][some].long()
    new = torch.where(cut, row, -1)
    new[some, tail[some]] = fresh.int()
    s["table"][kids] = new
    s["lens_now"][kids] = n.int()
    s["refs"].index_add_(0, new.clamp(min=0).view(-1).long(), (new.view(-1) >= 0).int())
    keep = (torch.arange(size, device="cuda") < slot[some][:, None])[:, None, None]
    for x in pages_out(s):
        keep_x = keep[..., None] if x.dim() == 5 else keep
        x[fresh] = torch.where(keep_x, x[old], x[fresh])
    return pages_out(s) + [s["table"], s["refs"], s["lens_now"]]


def plain_compact(s):
    """The k-th page in use behind the first n_live moves to the k-th free one among them."""
    live = s["refs_then"] > 0
    at = torch.arange(s["n_pages"], device="cuda")
    front = at < live.sum()
    src, dst = (live & ~front).nonzero().view(-1), (~live & front).nonzero().view(-1)
    for x in pages_out(s):
        x[dst] = x[src]
    to = at.int()
    to[src] = dst.int()
    s["table"].copy_(torch.where(s["table_then"] >= 0, to[s["table_then"].clamp(min=0).long()], -1))
    s["refs"].copy_(s["refs_then"])
    s["refs"][dst] = s["refs_then"][src]
    s["refs"][src] = 0
    return pages_out(s) + [s["table"], s["refs"]]


# ---------------------------------------------------------------------------
# The definition, in 64 bits
# ---------------------------------------------------------------------------
def attend(q, k, v, sees, scale):
    """Rows q [n][d] over entries k, v [m][d]; row i sees the first sees[i]."""
    x = (q @ k.T) * scale
    x = torch.where(torch.arange(k.shape[0], device=q.device) < sees[:, None], x, -math.inf)
    e = torch.exp(x - x.amax(1, keepdim=True))
    return torch.nan_to_num((e @ v) / e.sum(1, keepdim=True), nan=0.0)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prompt":
        return exact_prompt(case, s)
    if case["op"] == "decode":
        return exact_decode(case, s)
    if case["op"] == "store":
        return exact_store(case, s)
    return None  # pages are moved, not computed


def exact_prompt(c, s):
    d, group = c["dim"], c["heads"] // c["kv_heads"]
    out = torch.zeros(s["n_tokens"], c["heads"] * d, dtype=torch.float64, device="cuda")
    off = s["offsets"].tolist()
    for a, b in zip(off, off[1:]):
        for h in range(c["heads"]):
            kv = slice(h // group * d, (h // group + 1) * d)
            for at in range(a, b, 2048):
                end = min(b, at + 2048)
                out[at:end, h * d:(h + 1) * d] = attend(
                    s["q"][at:end, h * d:(h + 1) * d].double(), s["k"][a:end, kv].double(), s["v"][a:end, kv].double(),
                    torch.arange(at - a + 1, end - a + 1, device="cuda"), s["scale"])
    return out


def exact_decode(c, s):
    r, d, group, layer = c["rows"], c["dim"], c["heads"] // c["kv_heads"], c["layers"] - 1
    out = torch.zeros(c["seqs"] * r, c["heads"], d, dtype=torch.float64, device="cuda")
    q = s["q"].double().view(-1, c["heads"], d)
    for b, n in enumerate(s["lens_now"].tolist()):
        pages = s["table"][b, :-(-n // c["page"])].long()
        for h in range(c["kv_heads"]):
            k, v = (s[x][pages, layer, h].reshape(-1, d)[:n].double() for x in ("k", "v"))
            if s["ks"] is not None:
                k, v = (x * s[y][pages, layer, h].reshape(-1, 1)[:n].double() for x, y in ((k, "ks"), (v, "vs")))
            heads = slice(h * group, (h + 1) * group)
            sees = torch.arange(n - r + 1, n + 1, device="cuda").repeat_interleave(group)
            out[b * r:(b + 1) * r, heads] = attend(q[b * r:(b + 1) * r, heads].reshape(-1, d), k, v, sees,
                                                   s["scale"]).view(r, group, d)
    return out.view(c["seqs"] * r, -1)


def exact_store(c, s):
    """The cache with the new rows in it; codes of 8 bits follow from the rounding of 32 and have no such value."""
    table, used, off = s["table"].tolist(), s["lens_now"].tolist(), s["offsets"].tolist()
    where = [(table[b][p // c["page"]], p % c["page"]) for b in range(c["seqs"])
             for p in range(used[b] - (off[b + 1] - off[b]), used[b])]
    page, slot = torch.tensor(where, device="cuda").T
    got = []
    for x, scale, new in (("k", "ks", "new_k"), ("v", "vs", "new_v")):
        rows = s[new].double().view(-1, c["kv_heads"], c["dim"])
        into = (s[x] if s["ks"] is None else s[scale]).double()
        if s["ks"] is not None:
            rows = rows.abs().amax(-1) / 127
            rows = torch.where(rows == 0, 1.0, rows)
        into[page, c["layers"] - 1, :, slot] = rows
        got.append(into)
    return got if s["ks"] is None else [None, None] + got


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def slot_bytes(c):
    """One position of one kv head: key and value, and their scales."""
    return 2 * c["dim"] * SIZE[c["cache"]] + (8 if c["cache"] == "i8" else 0)


def work(case):
    c, op = case, case["op"]
    if op == "prompt":
        n = lengths(c, c["seqs"], c["shortest"], c["longest"])
        pairs = sum(x * (x + 1) // 2 for x in n)
        return {"bytes": sum(n) * 2 * (c["heads"] + c["kv_heads"]) * c["dim"] * SIZE[c["type"]] + 4 * (c["seqs"] + 1),
                "flops": 4 * pairs * c["heads"] * c["dim"]}
    if op == "store":
        new = sum(lengths(c, c["seqs"], c["fewest"], c["most"]))
        return {"bytes": new * c["kv_heads"] * (2 * c["dim"] * SIZE[c["type"]] + slot_bytes(c)),
                "flops": 4 * new * c["kv_heads"] * c["dim"]}
    if op == "decode":
        n = sum(lengths(c, c["seqs"], c["shortest"], c["longest"]))
        q = c["seqs"] * c["rows"] * c["heads"] * c["dim"]
        return {"bytes": n * c["kv_heads"] * slot_bytes(c) + 2 * q * SIZE[c["type"]] + 4 * pages_of(c, [n]),
                "flops": 4 * n * c["rows"] * c["heads"] * c["dim"]}
    slot = c["layers"] * c["kv_heads"] * slot_bytes(c)
    if op == "fork":
        n = fork_lens(c)
        tails = sum(x % c["page"] for x in n)
        rows = pages_of(c, n) * 4
        return {"bytes": tails * slot * (1 + c["fan"]) + rows * (1 + 2 * c["fan"]) + 4 * (pages_of(c, n) + c["spare"]),
                "flops": 0}
    n, table, refs = compact_layout(c)
    live = sum(x > 0 for x in refs)
    moved = sum(x > 0 for x in refs[live:])
    return {"bytes": 2 * moved * c["page"] * slot + 8 * c["pages"] + 8 * pages_of(c, n), "flops": 0}
