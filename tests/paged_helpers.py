"""A paged cache in torch tensors, the operators' definitions in 64 bits, and
the calls of the C ABI, for the paged cache's tests."""
import ctypes as C
import math
import random

import torch

from pocketforge_b200 import _lib

TYPES = {_lib.PF_F32: torch.float32, _lib.PF_BF16: torch.bfloat16, _lib.PF_F16: torch.float16, _lib.PF_I8: torch.int8}
F32, BF16, F16, I8 = _lib.PF_F32, _lib.PF_BF16, _lib.PF_F16, _lib.PF_I8


def ok(name, *args):
    _lib.check(getattr(_lib.lib(), name)(*args), name)


def stream():
    return torch.cuda.current_stream().cuda_stream


def latched(clear=True):
    """The device's error bits, cleared."""
    f = C.c_uint32()
    ok("pf_read_device_error", C.byref(f), 1 if clear else 0)
    return f.value


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Cache:
    def __init__(self, dtype=I8, layers=1, kv_heads=2, dim=64, page=16, pages=64, seqs=8, max_pages=16, fill=True,
                 seed=0):
        self.dtype, self.layers, self.kv_heads, self.dim, self.page = dtype, layers, kv_heads, dim, page
        self.pages, self.seqs, self.max_pages = pages, seqs, max_pages
        shape = (pages, layers, kv_heads, page)
        g = torch.Generator("cuda").manual_seed(seed)
        t = TYPES[dtype]
        self.ks = self.vs = None
        if not fill:
            self.k, self.v = (torch.empty((*shape, dim), dtype=t, device="cuda") for _ in range(2))
        elif dtype == I8:
            self.k, self.v = (torch.randint(-127, 128, (*shape, dim), generator=g, device="cuda", dtype=t)
                              for _ in range(2))
        else:
            self.k, self.v = (torch.randn((*shape, dim), generator=g, device="cuda").to(t) for _ in range(2))
        if dtype == I8:
            self.ks, self.vs = (torch.rand(shape, generator=g, device="cuda") * 0.01 + 0.01 for _ in range(2))
        self.table = torch.full((seqs, max_pages), -1, dtype=torch.int32, device="cuda")
        self.lens, self.refs = ints([0] * seqs), ints([0] * pages)
        p = lambda x: None if x is None else x.data_ptr()  # noqa: E731
        self.c = _lib.PagedCacheC(dtype=dtype, n_layers=layers, n_kv_heads=kv_heads, head_dim=dim, page_size=page,
                                  n_pages=pages, max_seqs=seqs, max_pages=max_pages, k=p(self.k), v=p(self.v),
                                  k_scale=p(self.ks), v_scale=p(self.vs), table=p(self.table), lens=p(self.lens),
                                  refs=p(self.refs))
        self.work = torch.zeros(_lib.lib().pf_paged_work_bytes(C.byref(self.c)), dtype=torch.uint8, device="cuda")
        self.c.work = p(self.work)
        self.ref = C.byref(self.c)
        self._alive = []

    def keep(self, *t):
        self._alive += t
        return [x.data_ptr() for x in t]

    def place(self, lens, seed=1):
        """Gives sequence b lens[b] tokens in pages taken in a random order."""
        order = random.Random(seed).sample(range(self.pages), self.pages)
        table, refs, at = self.table.tolist(), [0] * self.pages, 0
        for b, n in enumerate(lens):
            for j in range(-(-n // self.page)):
                table[b][j] = order[at]
                refs[order[at]] = 1
                at += 1
        self.table.copy_(ints(table))
        self.lens.copy_(ints(list(lens) + [0] * (self.seqs - len(lens))))
        self.refs.copy_(ints(refs))
        return self

    # ---- calls ----
    def reserve(self, seqs, counts):
        ok("pf_paged_reserve", self.ref, *self.keep(ints(seqs), ints(counts)), len(seqs), stream())

    def free(self, seqs):
        ok("pf_paged_free", self.ref, *self.keep(ints(seqs)), len(seqs), stream())

    def fork(self, parents, children):
        ok("pf_paged_fork", self.ref, *self.keep(ints(parents), ints(children)), len(parents), stream())

    def copy(self, src, dst):
        ok("pf_paged_copy", self.ref, *self.keep(ints(src), ints(dst)), len(src), stream())

    def compact(self):
        ok("pf_paged_compact", self.ref, stream())

    def store(self, layer, k, v, offsets, dtype, n_tokens=None):
        off = ints(offsets)
        ok("pf_paged_store", self.ref, layer, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), dtype,
           *self.keep(off), len(offsets) - 1, k.shape[0] if n_tokens is None else n_tokens, stream())

    def work_for(self, n_seqs, rows, heads):
        n = _lib.lib().pf_paged_attention_work_bytes(self.ref, n_seqs, rows, heads)
        assert n > 0
        return torch.zeros(n, dtype=torch.uint8, device="cuda")

    def attend(self, layer, q, out, dtype, n_seqs, rows, heads, scale, work=None):
        work = self.work_for(n_seqs, rows, heads) if work is None else work
        self.keep(work)
        ok("pf_paged_attention", self.ref, layer, q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), dtype,
           n_seqs, rows, heads, scale, work.data_ptr(), work.numel(), stream())

    # ---- the definitions ----
    def history(self, b, layer, g, n=None):
        """Keys and values of the first n positions of sequence b, in 64 bits."""
        n = int(self.lens[b]) if n is None else n
        pages = self.table[b, :-(-n // self.page)].long()
        k, v = (x[pages, layer, g].reshape(-1, self.dim)[:n].double() for x in (self.k, self.v))
        if self.ks is not None:
            k = k * self.ks[pages, layer, g].reshape(-1, 1)[:n].double()
            v = v * self.vs[pages, layer, g].reshape(-1, 1)[:n].double()
        return k, v

    def attention(self, layer, q, n_seqs, rows, heads, scale):
        """(out, tolerance's parts: largest |v|, largest sum |q||k| scale) of the definition, [tokens][heads][dim]."""
        q = q.double().view(n_seqs * rows, heads, self.dim)
        out = torch.zeros_like(q)
        big_v, big_s = torch.zeros(q.shape[:2] + (1,), device="cuda").double(), torch.zeros_like(q[..., :1])
        for b in range(n_seqs):
            n = int(self.lens[b])
            for h in range(heads):
                k, v = self.history(b, layer, h // (heads // self.kv_heads))
                for r in range(rows):
                    m = n - rows + 1 + r
                    if m <= 0:
                        continue
                    out[b * rows + r, h] = softmax_mean(q[b * rows + r, h] @ k[:m].T * scale, v[:m])
                    big_v[b * rows + r, h] = v[:m].abs().max()
                    big_s[b * rows + r, h] = (q[b * rows + r, h].abs() @ k[:m].abs().T * scale).max()
        return out, big_v, big_s


def softmax_mean(x, v):
    e = torch.exp(x - x.max())
    return (e / e.sum()) @ v


def prompt(q, k, v, offsets, heads, kv_heads, dim, scale):
    """The prompt attention's definition in 64 bits, and its tolerance's parts, as Cache.attention gives them."""
    n = q.shape[0]
    out = torch.full((n, heads, dim), math.nan, dtype=torch.float64, device="cuda")
    big_v, big_s = torch.zeros(n, heads, 1, device="cuda").double(), torch.zeros(n, heads, 1, device="cuda").double()
    for a, e in zip(offsets, offsets[1:]):
        causal = torch.ones(e - a, e - a, device="cuda").tril().bool()
        for h in range(heads):
            g = h // (heads // kv_heads)
            qq, kk, vv = (x[a:e, i * dim:(i + 1) * dim].double() for x, i in ((q, h), (k, g), (v, g)))
            if e == a:
                continue
            x = torch.where(causal, qq @ kk.T * scale, -math.inf)
            p = torch.exp(x - x.amax(1, keepdim=True))
            out[a:e, h] = (p / p.sum(1, keepdim=True)) @ vv
            big_v[a:e, h] = torch.cummax(vv.abs().amax(1), 0).values[:, None]
            big_s[a:e, h] = torch.where(causal, qq.abs() @ kk.abs().T * scale, 0.0).amax(1, keepdim=True)
    return out, big_v, big_s


def tolerance(t, out, big_v, big_s):
    """How far an output of type t may be from the definition's.

    A score is a sum of up to 128 products whose operands carry 22 bits or
    more (2^-22 of each product) and whose sums are rounded or cut to 24 bits
    at each of at most 16 steps (16 x 2^-23): off by 2^-18 of sum |q||k| scale
    at most, its weight by twice that, and by 2^-20 for the exponential and the
    row's sum.  The weights average values of at most big_v.  16-bit outputs:
    the weights may be rounded to the type (eps / 2 of each, so eps / 2 of
    big_v) and the output is (eps / 2 of itself); fp16 weights below its normal
    range are off by 2^-25 absolutely, which 2^-18 of big_v covers up to 128
    of them against a row sum of at least 1 ... the rest of a longer row is
    covered because each such weight is itself below 2^-14.
    """
    f32 = (2.0 ** -17 * big_s + 2.0 ** -18) * big_v
    if t == torch.float32:
        return f32 + 2.0 ** -24 * out.abs()
    half = torch.finfo(t).eps / 2
    return f32 + half * big_v + half * out.abs()


def check(got, want, t):
    out, big_v, big_s = want
    d = (got.double().view_as(out) - out).abs()
    tol = tolerance(t, out, big_v, big_s)
    assert not torch.isnan(d).any(), "NaN where the definition has none"
    worst = (d - tol).max()
    assert worst <= 0, f"off by {d.max():.3g}, {(d / tol.clamp(min=1e-300)).max():.3g} of the tolerance"
