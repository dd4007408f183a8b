"""Operators of continuous batching over an 8-bit paged K/V cache, and what they cost.

Four operators that a serving loop runs one after another:

  plan    block tables, row maps and slot maps of one step, from request lengths
          (wk_batch_plan)
  store   K and V rows quantised to e4m3 into the pages of the cache, one power
          of two per page and K/V head as the scale (wk_kv8_store)
  decode  attention of single tokens over that cache (wk_kv8_attention)
  prompt  causal attention with grouped heads over packed sequences
          (wk_attention_packed)

`own` false: the plain form in elementary torch operations.  `own` true: the
library's entry points.
"""
import math

import torch

own = False

PAGE = 64
F16, BF16 = 1, 30  # GGML type ids
DT = {"f16": (torch.float16, F16), "bf16": (torch.bfloat16, BF16)}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
MIN_EXP = -100  # scale exponent of a page that holds zeros only


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # the map of one decode step: 64 running sequences, one token each
        dict(name="plan_step_64", op="plan", n=64, grow=1, prompts=0, ctx_max=8192, max_pages=256),
        # a busy step: 500 running sequences and 12 prompts of up to 2048 tokens that join
        dict(name="plan_mixed_512", op="plan", n=512, grow=1, prompts=12, ctx_max=16384, max_pages=512),
        # one token of each of 48 sequences appended to an 8 x 128 cache
        dict(name="store_step_48", op="store", n=48, add_lo=1, add_hi=1, ctx_max=4096, heads=32, kv_heads=8, hd=128,
             dt="f16"),
        # packed prompts of odd lengths, most of them behind a context that ends inside a page
        dict(name="store_prompts", op="store", n=9, add_lo=301, add_hi=2303, ctx_max=999, heads=32, kv_heads=8,
             hd=128, dt="bf16"),
        # the smallest call: one sequence, a short context, 16 query heads of 64
        dict(name="decode_1x777", op="decode", rows=1, len_lo=777, len_hi=777, heads=16, kv_heads=4, hd=64, dt="f16"),
        # an ordinary batch: ragged contexts, the 8B head layout
        dict(name="decode_64_ragged", op="decode", rows=64, len_lo=130, len_hi=8191, heads=32, kv_heads=8, hd=128,
             dt="f16"),
        # the 70B head layout, 8 query heads per K/V head
        dict(name="decode_16x4096", op="decode", rows=16, len_lo=3500, len_hi=4096, heads=64, kv_heads=8, hd=128,
             dt="bf16"),
        # one rank of eight of that model, a single very long context
        dict(name="decode_1x131071", op="decode", rows=1, len_lo=131071, len_hi=131071, heads=8, kv_heads=1, hd=128,
             dt="bf16"),
        # one short question
        dict(name="prompt_1x97", op="prompt", n=1, lo=97, hi=97, before=0, heads=32, kv_heads=8, hd=128, dt="f16"),
        # prompts of many lengths packed into one step, heads of 64
        dict(name="prompt_24_ragged", op="prompt", n=24, lo=1, hi=1500, before=0, heads=16, kv_heads=4, hd=64,
             dt="f16"),
        # a long prompt, the 8B head layout
        dict(name="prompt_1x8192", op="prompt", n=1, lo=8192, hi=8192, before=0, heads=32, kv_heads=8, hd=128,
             dt="bf16"),
        # the last chunk of a long document on one rank of eight: 2000 new rows behind 14000 tokens
        dict(name="prompt_chunk", op="prompt", n=1, lo=2000, hi=2000, before=14000, heads=8, kv_heads=1, hd=128,
             dt="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["plan", "store", "decode", "prompt"])
    dt = rng.choice(["f16", "bf16"])
    hd = rng.choice([64, 128])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 5, 7, 8, 16] if kv < 8 else [1, 2, 4, 5, 8])
    if op == "plan":
        n = _log(rng, 1, 1000)
        return dict(op=op, n=n, grow=rng.choice([1, 1, 1, 5]), prompts=rng.randint(0, min(n, 12)),
                    ctx_max=_log(rng, 10, 16000), max_pages=rng.choice([300, 411, 512]))
    if op == "store":
        step = rng.random() < 0.5
        n = _log(rng, 1, 256) if step else _log(rng, 1, 16)
        hi = 1 if step else _log(rng, 2, 10000 // n)
        return dict(op=op, n=n, add_lo=1 if step else rng.randint(1, hi), add_hi=hi, ctx_max=_log(rng, 1, 3000),
                    heads=heads, kv_heads=kv, hd=hd, dt=dt)
    if op == "decode":
        rows = _log(rng, 1, 64)
        hi = _log(rng, 1, min(100000, 1000000 // (rows * kv)))
        return dict(op=op, rows=rows, len_lo=rng.randint(1, hi), len_hi=hi, heads=heads, kv_heads=kv, hd=hd, dt=dt)
    n = _log(rng, 1, 24)
    most = int(math.sqrt(8192 * 8192 * 32 / 4 / (n * heads)))
    hi = _log(rng, 1, min(6000, most))
    before = rng.choice([0, 0, rng.randint(1, max(1, min(4000, most)))])
    return dict(op=op, n=n, lo=rng.randint(1, hi), hi=hi, before=before, heads=heads, kv_heads=kv, hd=hd, dt=dt)


# ------------------------------------------------------------------ the inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _spread(n, lo, hi):
    """n lengths of [lo, hi], the first hi and the others spread over the logarithm: the same for every seed."""
    golden = (math.sqrt(5) - 1) / 2
    return [hi] + [min(hi, int(lo * ((hi + 0.999) / lo) ** (i * golden % 1))) for i in range(1, n)]


def _lengths(n, lo, hi, g):
    """Those lengths in an order of this seed."""
    v = torch.tensor(_spread(n, lo, hi), dtype=torch.int32, device="cuda")
    return v[torch.randperm(n, generator=g, device="cuda")]


def _adds(c):
    """What each sequence of a plan brings: the prompts first, then a few tokens each."""
    p, n = c["prompts"], c["n"]
    return (_spread(p, 16, 2048) if p else []) + (_spread(n - p, 1, c["grow"]) if n > p else [])


def _starts(lens):
    return torch.cat([lens.new_zeros(1), torch.cumsum(lens, 0, dtype=torch.int32)])


def _int32(*shape, fill=0):
    return torch.full(shape, fill, dtype=torch.int32, device="cuda")


def _random_cache(n_pages, kv, hd, g):
    """Pages as earlier steps left them: e4m3 codes of normal values, a power of two per page and head."""
    codes, scales = [], []
    for _ in range(2):
        x = torch.randn(n_pages, kv, PAGE, hd, generator=g, device="cuda", dtype=torch.float16)
        e = torch.randint(-9, -5, (n_pages, kv), generator=g, device="cuda", dtype=torch.int32)
        x.mul_(torch.randint(40, 110, (n_pages, kv, 1, 1), generator=g, device="cuda", dtype=torch.int32).half())
        codes.append(x.clamp_(-E4M3_MAX, E4M3_MAX).to(E4M3).view(torch.uint8))
        scales.append(torch.ldexp(torch.ones(n_pages, kv, device="cuda"), e))
    return codes[0], codes[1], scales[0], scales[1]


def _tables(pages_of, max_pages, n_pages, g):
    """Block tables over a shuffled pool: sequence i has its pages_of[i] first entries, the others are -1."""
    n = pages_of.numel()
    p = torch.arange(max_pages, device="cuda", dtype=torch.int32)[None, :]
    base = (torch.cumsum(pages_of, 0) - pages_of)[:, None]
    perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    idx = (base + p).clamp(0, n_pages - 1).long()
    return torch.where(p < pages_of[:, None], perm[idx], torch.full((n, max_pages), -1, dtype=torch.int32,
                                                                   device="cuda"))


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = dict(c)
    if c["op"] == "plan":
        n = c["n"]
        ctx = _lengths(n, 1, c["ctx_max"], g)
        at = torch.randperm(n, generator=g, device="cuda")
        add = torch.empty_like(ctx)
        add[at] = torch.tensor(_adds(c), dtype=torch.int32, device="cuda")
        ctx[at[: c["prompts"]]] = 0
        have = (ctx + PAGE - 1) // PAGE
        new = (ctx + add + PAGE - 1) // PAGE - have
        held, taken = int(have.sum()), int(new.sum())
        n_free = taken + 50
        n_pages = held + n_free
        perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        s["table"] = _tables(have, c["max_pages"], n_pages, g)
        s.update(ctx=ctx, add=add, free=perm[:n_free].contiguous(), n_free=_int32(1, fill=n_free), cap=int(add.sum()) + 7)
        cap = s["cap"]
        s.update(starts=_int32(n + 1), lens=_int32(n), row_seq=_int32(cap), row_pos=_int32(cap),
                 row_slot=torch.zeros(cap, dtype=torch.int64, device="cuda"), status=_int32(3))
    elif c["op"] == "store":
        n, kv, hd = c["n"], c["kv_heads"], c["hd"]
        add = _lengths(n, c["add_lo"], c["add_hi"], g)
        ctx = torch.randint(0, c["ctx_max"] + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
        rows = int(add.sum())
        pages_of = (ctx + add + PAGE - 1) // PAGE
        s["n_pages"] = sum((c["ctx_max"] + a + PAGE - 1) // PAGE for a in _spread(n, c["add_lo"], c["add_hi"])) + 5
        s["max_pages"] = int(pages_of.max()) + 1
        s["table"] = _tables(pages_of, s["max_pages"], s["n_pages"], g)
        s["kpool"], s["vpool"], s["kscale"], s["vscale"] = _random_cache(s["n_pages"], kv, hd, g)
        # rows as the q|k|v projection writes them; a few sequences outgrow the scale of their open page
        w = (c["heads"] + 2 * kv) * hd
        qkv = torch.randn(rows, w, generator=g, device="cuda", dtype=torch.float32)
        grow = torch.exp2(torch.randint(-1, 3, (rows, 1), generator=g, device="cuda").float())
        qkv = (qkv * grow).to(DT[c["dt"]][0])
        s.update(qkv=qkv, k=qkv[:, c["heads"] * hd:(c["heads"] + kv) * hd], v=qkv[:, (c["heads"] + kv) * hd:],
                 starts=_starts(add), ctx=ctx, nrows=rows)
    elif c["op"] == "decode":
        rows, kv, hd, h = c["rows"], c["kv_heads"], c["hd"], c["heads"]
        lens = _lengths(rows, c["len_lo"], c["len_hi"], g)
        pages_of = (lens + PAGE - 1) // PAGE
        s["n_pages"] = int(pages_of.sum()) + 3
        s["max_pages"] = int(pages_of.max())
        s["table"] = _tables(pages_of, s["max_pages"], s["n_pages"], g)
        s["kpool"], s["vpool"], s["kscale"], s["vscale"] = _random_cache(s["n_pages"], kv, hd, g)
        dt = DT[c["dt"]][0]
        s.update(q=torch.randn(rows, h * hd, generator=g, device="cuda").to(dt), pos=lens - 1,
                 seq=torch.arange(rows, device="cuda", dtype=torch.int32),
                 out=torch.zeros(rows, h * hd, dtype=dt, device="cuda"))
        # the workspace that a serving program keeps: the partial sums of a split context
        s["ws"] = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    else:
        n, kv, hd, h = c["n"], c["kv_heads"], c["hd"], c["heads"]
        ql = _lengths(n, c["lo"], c["hi"], g)
        kl = ql + c["before"]
        tq, tk = int(ql.sum()), int(kl.sum())
        dt = DT[c["dt"]][0]
        if c["before"]:
            s["q"] = torch.randn(tq, h * hd, generator=g, device="cuda").to(dt)
            kvrows = torch.randn(tk, 2 * kv * hd, generator=g, device="cuda").to(dt)
            s["k"], s["v"] = kvrows[:, : kv * hd], kvrows[:, kv * hd:]
        else:  # q|k|v rows as the projection writes them
            rows = torch.randn(tq, (h + 2 * kv) * hd, generator=g, device="cuda").to(dt)
            s["q"], s["k"], s["v"] = rows[:, : h * hd], rows[:, h * hd:(h + kv) * hd], rows[:, (h + kv) * hd:]
        s.update(q_starts=_starts(ql), k_starts=_starts(kl), q_rows=tq, k_rows=tk, q_max=int(ql.max()),
                 k_max=int(kl.max()), out=torch.zeros(tq, h * hd, dtype=dt, device="cuda"))
    return s


# ------------------------------------------------------------------ plain forms

def _plan(s):
    """The maps of a step: sequence i brings add[i] tokens behind ctx[i]; new pages come from the free list in order."""
    ctx, add, n, cap = s["ctx"].long(), s["add"].long(), s["n"], s["cap"]
    starts = torch.cat([add.new_zeros(1), torch.cumsum(add, 0)])
    have, need = (ctx + PAGE - 1) // PAGE, (ctx + add + PAGE - 1) // PAGE
    need = torch.maximum(have, need.clamp(max=s["max_pages"]))
    base = torch.cumsum(need - have, 0) - (need - have)
    p = torch.arange(s["max_pages"], device="cuda")[None, :]
    i = base[:, None] + p - have[:, None]
    page = torch.where(i < s["n_free"], s["free"][i.clamp(0, s["free"].numel() - 1)], -1)
    s["table"].copy_(torch.where((p >= have[:, None]) & (p < need[:, None]), page, s["table"]))
    r = torch.arange(cap, device="cuda")
    seq = torch.searchsorted(starts[1:], r, right=True)
    real = seq < n
    seq = seq.clamp(max=n - 1)
    pos = r - starts[seq] + ctx[seq]
    at = s["table"][seq, (pos // PAGE).clamp(max=s["max_pages"] - 1)].long()
    slot = torch.where((at >= 0) & (pos < PAGE * s["max_pages"]), at * PAGE + pos % PAGE, -1)
    want = (need - have).sum()
    taken = torch.minimum(want, s["n_free"][0])
    return {"starts": starts.int(), "lens": (ctx + add).int(), "row_seq": torch.where(real, seq, -1).int(),
            "row_pos": torch.where(real, pos, -1).int(), "row_slot": torch.where(real, slot, -1), "table": s["table"],
            "status": torch.stack([starts[-1], taken, want - taken]).int()}


def _scale_of(amax):
    """The smallest power of two s with amax <= 448 s (448 = 0.875 * 2^9)."""
    f, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - 9 + (f > 0.875).to(e.dtype), MIN_EXP).clamp(min=MIN_EXP)
    return torch.ldexp(torch.ones_like(amax), e)


def _store_one(pool, scale, x, page, off, kv, hd):
    x = x.float().reshape(x.shape[0], kv, hd)
    # what the call needs of each page's scale, and the first place that it writes there
    touched, inv = torch.unique(page, return_inverse=True)
    need = _scale_of(torch.zeros(touched.numel(), kv, device="cuda").index_reduce_(0, inv, x.abs().amax(2), "amax"))
    first = torch.full((touched.numel(),), PAGE, device="cuda", dtype=torch.long).scatter_reduce_(0, inv, off, "amin")
    old = scale[touched]
    new = torch.where(first[:, None] > 0, torch.maximum(old, need), need)
    # tokens that the page held before keep their values, in steps of the new scale
    held = pool[touched]
    again = (held.view(E4M3).float() * (old / new)[:, :, None, None]).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3)
    keep = torch.arange(PAGE, device="cuda")[None, :] < first[:, None]
    pool[touched] = torch.where(keep[:, None, :, None], again.view(torch.uint8), held)
    scale[touched] = new
    code = (x / new[inv][:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3).view(torch.uint8)
    pool[page, :, off] = code


def _store(s):
    r = torch.arange(s["nrows"], device="cuda")
    starts = s["starts"].long()
    seq = torch.searchsorted(starts[1:], r, right=True)
    pos = r - starts[seq] + s["ctx"].long()[seq]
    page, off = s["table"][seq, pos // PAGE].long(), pos % PAGE
    _store_one(s["kpool"], s["kscale"], s["k"], page, off, s["kv_heads"], s["hd"])
    _store_one(s["vpool"], s["vscale"], s["v"], page, off, s["kv_heads"], s["hd"])


def _softmax(scores, seen):
    """Softmax over the last axis among the places seen; zeros where a row sees none."""
    scores = scores.masked_fill_(~seen, -math.inf)
    m = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    return p.div_(p.sum(-1, keepdim=True).clamp(min=torch.finfo(p.dtype).tiny))


def _decode(s):
    rows, h, kv, hd = s["rows"], s["heads"], s["kv_heads"], s["hd"]
    table = s["table"][s["seq"].long()].long().clamp(min=0)
    k = s["kpool"][table].view(E4M3).float().mul_(s["kscale"][table][..., None, None])  # [rows, pages, kv, 64, hd]
    k = k.permute(0, 2, 1, 3, 4).reshape(rows, kv, -1, hd)
    q = s["q"].float().reshape(rows, kv, h // kv, hd) / math.sqrt(hd)
    scores = torch.matmul(q, k.transpose(2, 3))
    del k
    seen = torch.arange(scores.shape[-1], device="cuda")[None, :] <= s["pos"][:, None]
    p = _softmax(scores, seen[:, None, None, :])
    v = s["vpool"][table].view(E4M3).float().mul_(s["vscale"][table][..., None, None])
    v = v.permute(0, 2, 1, 3, 4).reshape(rows, kv, -1, hd)
    return torch.matmul(p, v).reshape(rows, h * hd).to(s["q"].dtype)


def _prompt(s):
    h, kv, hd, n = s["heads"], s["kv_heads"], s["hd"], s["n"]
    qs, ks = s["q_starts"].long(), s["k_starts"].long()
    ql, kl = qs[1:] - qs[:-1], ks[1:] - ks[:-1]
    i = torch.arange(s["q_max"], device="cuda")[None, :]
    j = torch.arange(s["k_max"], device="cuda")[None, :]
    qi = (qs[:-1, None] + i).clamp(max=s["q_rows"] - 1)
    kj = (ks[:-1, None] + j).clamp(max=s["k_rows"] - 1)
    q = s["q"][qi].float().reshape(n, -1, kv, h // kv, hd).permute(0, 2, 3, 1, 4) / math.sqrt(hd)
    k = s["k"][kj].float().reshape(n, -1, kv, hd).permute(0, 2, 3, 1)
    v = s["v"][kj].float().reshape(n, -1, kv, hd).permute(0, 2, 1, 3)
    at = i + (kl - ql)[:, None]  # the position of each query among its sequence's keys
    seen = (j[:, None, :] <= at[:, :, None]) & (j < kl[:, None])[:, None, :]
    p = _softmax(torch.matmul(q, k[:, :, None]), seen[:, None, None])
    o = torch.matmul(p, v[:, :, None]).permute(0, 3, 1, 2, 4).reshape(n, -1, h * hd)
    return o[(i < ql[:, None])].to(s["q"].dtype)


# ------------------------------------------------------------------ the library's calls

_L = None


def _lib():
    """The library on device 0; torch works on the library's stream from then on, so that the two are ordered."""
    global _L
    if _L is None:
        import wukong_b200 as wk
        _L = wk.lib()
        _L.cuda_init(0)
        torch.cuda.set_stream(torch.cuda.ExternalStream(_L.wk_stream()))
    return _L


def _own(s):
    lib = _lib()
    p = lambda name: s[name].data_ptr()  # noqa: E731
    if s["op"] == "plan":
        rc = lib.wk_batch_plan(p("starts"), p("lens"), p("row_seq"), p("row_pos"), p("row_slot"), s["cap"], p("table"),
                               s["max_pages"], p("status"), p("ctx"), p("add"), s["n"], p("free"), p("n_free"),
                               s["free"].numel())
        out = {k: s[k] for k in ("starts", "lens", "row_seq", "row_pos", "row_slot", "table", "status")}
    elif s["op"] == "store":
        rc = lib.wk_kv8_store(p("kpool"), p("vpool"), p("kscale"), p("vscale"), s["n_pages"], p("k"), s["k"].stride(0),
                              p("v"), s["v"].stride(0), p("starts"), p("ctx"), s["n"], s["nrows"], p("table"),
                              s["max_pages"], s["kv_heads"], s["hd"], DT[s["dt"]][1])
        out = _cache_of(s)
    elif s["op"] == "decode":
        rc = lib.wk_kv8_attention(p("out"), s["out"].stride(0), p("q"), s["q"].stride(0), p("kpool"), p("vpool"),
                                  p("kscale"), p("vscale"), s["n_pages"], p("table"), s["table"].shape[0],
                                  s["max_pages"], p("seq"), p("pos"), s["rows"], s["len_hi"], s["heads"],
                                  s["kv_heads"], s["hd"], DT[s["dt"]][1], p("ws"), s["ws"].numel())
        out = s["out"]
    else:
        rc = lib.wk_attention_packed(p("out"), s["out"].stride(0), p("q"), s["q"].stride(0), p("k"), s["k"].stride(0),
                                     p("v"), s["v"].stride(0), p("q_starts"), p("k_starts"), s["n"], s["q_rows"],
                                     s["k_rows"], s["heads"], s["kv_heads"], s["hd"], DT[s["dt"]][1])
        out = s["out"]
    if rc != 0:
        raise RuntimeError(lib.wk_last_error().decode())
    return out


def _cache_of(s):
    return {"k": s["kpool"].view(E4M3), "v": s["vpool"].view(E4M3), "kscale": s["kscale"], "vscale": s["vscale"]}


def run(state):
    if own:
        return _own(state)
    if state["op"] == "plan":
        return _plan(state)
    if state["op"] == "store":
        _store(state)
        return _cache_of(state)
    return _decode(state) if state["op"] == "decode" else _prompt(state)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    c = case
    if c["op"] == "plan":
        rows = sum(_adds(c))
        # request lengths in, starts and lengths out, 16 bytes of maps per row; new table entries in and out
        return {"bytes": 16 * c["n"] + 16 * rows + 8 * (rows // PAGE + 1), "flops": 0}
    if c["op"] == "store":
        adds = _spread(c["n"], c["add_lo"], c["add_hi"])
        # 16-bit rows in, 8-bit rows out, the scales of the pages in and out
        pages = sum(a // PAGE + 1 for a in adds)
        return {"bytes": 6 * sum(adds) * c["kv_heads"] * c["hd"] + 16 * pages * c["kv_heads"], "flops": 0}
    if c["op"] == "decode":
        keys = sum(_spread(c["rows"], c["len_lo"], c["len_hi"]))
        return {"bytes": 2 * keys * c["kv_heads"] * (c["hd"] + 4 / PAGE) + 4 * c["rows"] * c["heads"] * c["hd"],
                "flops": 4 * keys * c["heads"] * c["hd"]}
    ql = _spread(c["n"], c["lo"], c["hi"])
    rows, keys = sum(ql), sum(ql) + c["n"] * c["before"]
    pairs = sum(a * (a + 1) // 2 + a * c["before"] for a in ql)
    return {"bytes": 4 * rows * c["heads"] * c["hd"] + 4 * keys * c["kv_heads"] * c["hd"],
            "flops": 4 * pairs * c["heads"] * c["hd"]}


# ------------------------------------------------------------------ the definitions in 64 bits

def _round_e4m3(y):
    """The nearest e4m3 value (ties to the even code) of a float64, saturating at 448."""
    a = y.abs().clamp(max=E4M3_MAX)
    exponent = torch.floor(torch.log2(a.clamp(min=2.0 ** -6)))
    exponent = exponent + (a >= torch.exp2(exponent + 1)) - (a < torch.exp2(exponent)).double() * (a >= 2.0 ** -6)
    step = torch.exp2(exponent - 3)
    return torch.sign(y) * torch.round(a / step) * step


def _exact_store(s):
    kv, hd = s["kv_heads"], s["hd"]
    ctx, starts, table = s["ctx"].tolist(), s["starts"].tolist(), s["table"].tolist()
    result = {}
    for name in ("k", "v"):
        codes, scale = s[name + "pool"].view(E4M3).double(), s[name + "scale"].double()
        x = s[name].double().reshape(-1, kv, hd)
        for q in range(s["n"]):
            row, pos, end = starts[q], ctx[q], ctx[q] + starts[q + 1] - starts[q]
            while pos < end:
                page, off = table[q][pos // PAGE], pos % PAGE
                m = min(PAGE - off, end - pos)
                block = x[row:row + m].permute(1, 0, 2)  # [kv, m, hd]
                top = block.abs().amax((1, 2))
                e = torch.ceil(torch.log2((top / E4M3_MAX).clamp(min=2.0 ** -300)))
                e = torch.where(top > E4M3_MAX * torch.exp2(e), e + 1, e)
                e = torch.where(top <= E4M3_MAX * torch.exp2(e - 1), e - 1, e).clamp(min=MIN_EXP)
                new = torch.exp2(e)
                if off:
                    new = torch.maximum(new, scale[page])
                    codes[page, :, :off] = _round_e4m3(codes[page, :, :off] * (scale[page] / new)[:, None, None])
                codes[page, :, off:off + m] = _round_e4m3(block / new[:, None, None])
                scale[page] = new
                row, pos = row + m, pos + m
        result[name], result[name + "scale"] = codes, scale
    return {k: result[k] for k in ("k", "v", "kscale", "vscale")}


def _attend(q, k, v, first):
    """softmax(q k^T / sqrt(d)) v, query i seeing the keys up to first + i: q [g, m, d], k and v [l, d], in 64 bits."""
    m, l = q.shape[1], k.shape[0]
    scores = q @ k.T / math.sqrt(q.shape[-1])
    hidden = torch.arange(l, device="cuda")[None, :] > torch.arange(m, device="cuda")[:, None] + first
    scores.masked_fill_(hidden, -math.inf)
    return torch.softmax(scores, -1) @ v


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None
    if case["op"] == "store":
        return _exact_store(s)
    h, kv, hd = s["heads"], s["kv_heads"], s["hd"]
    g = h // kv
    if case["op"] == "decode":
        out = torch.zeros(s["rows"], h, hd, dtype=torch.float64, device="cuda")
        for r, p in enumerate(s["pos"].tolist()):
            pages = s["table"][r, : p // PAGE + 1].long()
            for a in range(kv):
                k, v = ((s[x + "pool"][pages, a].view(E4M3).double() * s[x + "scale"][pages, a].double()[:, None, None])
                        .reshape(-1, hd)[: p + 1] for x in "kv")
                q = s["q"][r].double().reshape(h, 1, hd)[a * g:(a + 1) * g]
                out[r, a * g:(a + 1) * g] = _attend(q, k, v, p)[:, 0]
        return out.reshape(s["rows"], h * hd)
    out = torch.zeros(s["q_rows"], h, hd, dtype=torch.float64, device="cuda")
    qs, ks = s["q_starts"].tolist(), s["k_starts"].tolist()
    for i in range(s["n"]):
        ql, kl = qs[i + 1] - qs[i], ks[i + 1] - ks[i]
        for a in range(kv):
            k, v = (s[x][ks[i]:ks[i + 1], a * hd:(a + 1) * hd].double() for x in "kv")
            for b in range(a * g, (a + 1) * g):
                q = s["q"][qs[i]:qs[i + 1], b * hd:(b + 1) * hd].double()
                out[qs[i]:qs[i + 1], b] = _attend(q[None], k, v, kl - ql)[0]
    return out.reshape(s["q_rows"], h * hd)
