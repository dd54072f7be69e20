"""The key / value cache in 4 bits, measured: writing it, decoding from it, prompts over it.

A page of one kv head holds ``block_size`` token rows of ``head_dim`` e2m1 numbers, two to a byte
(even element in the low half), and behind them the rows' scales: one power of two, as a byte
(exponent + 127), for every 32 elements of a row.  Caches are uint8 tensors
[pages, kv heads, block_size, head_dim / 2 + head_dim / 32]; the last two dimensions are one page:
block_size * head_dim / 2 bytes of numbers, then block_size * head_dim / 32 scales.

  write    q, k, v of a step from its QKV projection: q and k rotated, k and v into their pages.  The
           pages' new rows are read back as the values they stand for.
  axes     the same where a token has a position on several axes (time, height, width): pair i of a
           head turns by the position of the axis that its section belongs to.
  decode   one query row per sequence against its cached tokens.
  prompts  a step's prompt rows, causally, against everything their sequences have cached.

Heads are those of the presets that the service runs (32 / 8 heads of 128), and 12 / 12 heads of 64.
``draw`` spreads over the same ranges: one row to 16384, contexts from one token to 32768.
"""
import math

import numpy as np
import torch

own = False

PAGE = 32                      # tokens per cache page: the engine's default
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}
HEADS = {                      # q heads, kv heads, head size
    "gqa": (32, 8, 128),       # Llama-3-8B, Mixtral
    "gqa8": (64, 8, 128),      # Llama-3-70B
    "tp8": (8, 1, 128),        # the same on one of eight GPUs
    "mha": (12, 12, 64),       # OPT-125m
}
SECTIONS = {128: (16, 24, 24), 64: (8, 12, 12)}    # pairs per axis: time, height, width
THETA = 500000.0
LUT = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)      # e2m1
# the scales' exponents: every value of a block is one of the activations' type
EXPONENTS = {torch.bfloat16: (-120, 125), torch.float16: (-22, 13)}


def listed():
    return [
        # a decode step of the service's full batch, some rows of it graph padding
        dict(name="write 256", kind="write", heads="gqa", dtype="bfloat16", rows=256, pad=9),
        # a full prefill step
        dict(name="write 16384", kind="write", heads="gqa", dtype="bfloat16", rows=16384, pad=0),
        # a prompt of text and one image, and of a long video
        dict(name="axes 1111", kind="axes", heads="gqa", dtype="float16", rows=1111, pad=0, cache="fp4"),
        dict(name="axes 12000", kind="axes", heads="gqa", dtype="bfloat16", rows=12000, pad=0, cache="auto"),
        # a single short request; the service's full batch; many long ones; one very long one;
        # small heads in fp16
        dict(name="decode 1x128", kind="decode", heads="gqa", dtype="bfloat16", seqs=1, ctx=128),
        dict(name="decode 256x640", kind="decode", heads="gqa", dtype="bfloat16", seqs=256, ctx=640),
        dict(name="decode 64x8192", kind="decode", heads="gqa", dtype="bfloat16", seqs=64, ctx=8192),
        dict(name="decode 1x32000", kind="decode", heads="gqa8", dtype="bfloat16", seqs=1, ctx=32000),
        dict(name="decode 33x1001 f16", kind="decode", heads="mha", dtype="float16", seqs=33, ctx=1001),
        # full prefill steps of short and of long prompts, a chunk that continues long prompts
        dict(name="prompts 32x512", kind="prompts", heads="gqa", dtype="bfloat16", seqs=32, len=512, ctx=0),
        dict(name="prompts 4x4096", kind="prompts", heads="gqa", dtype="bfloat16", seqs=4, len=4096, ctx=0),
        dict(name="prompts 3x301 after 7000", kind="prompts", heads="mha", dtype="float16", seqs=3, len=301, ctx=7000),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "axes", "decode", "decode", "prompts", "prompts"])
    c = dict(kind=kind, heads=rng.choice(["gqa", "gqa", "gqa8", "tp8", "mha"]),
             dtype=rng.choice(["bfloat16", "bfloat16", "float16"]))
    nq, nkv, d = HEADS[c["heads"]]
    if kind in ("write", "axes"):
        c["rows"] = _log(rng, 1, 16384 if kind == "write" else 12000)
        if nq > 32:
            c["rows"] = max(1, c["rows"] // 2)
        c["pad"] = rng.choice([0, min(c["rows"] // 4, 15)])
        if kind == "axes":
            c["cache"] = rng.choice(["fp4", "fp4", "auto"])
    elif kind == "decode":
        c["seqs"] = _log(rng, 1, 256)
        # no more cached elements than 64 x 8192 tokens of 8 heads of 128 have
        most = min(32768, 64 * 8192 * 8 * 128 // (c["seqs"] * nkv * d), 64 * 8192 * 32 * 128 // (c["seqs"] * nq * d))
        c["ctx"] = _log(rng, 1, most)
    else:
        c["len"] = _log(rng, 1, 4096)
        c["seqs"] = _log(rng, 1, max(1, min(64, 16384 // c["len"])))
        c["ctx"] = rng.choice([0, 0, _log(rng, 1, 8192)])
        most = _flops(dict(kind="prompts", heads="gqa", seqs=4, len=4096, ctx=0))
        while _flops(c) > most:
            if c["seqs"] > 1:
                c["seqs"] //= 2
            else:
                c["ctx"] //= 2
    return c


# ------------------------------------------------------------------ shapes of a case
def _lens(n, base):
    """Ragged lengths: the first is ``base``, the others down to three quarters of it."""
    return [base - (i * 37) % (base // 4 + 1) for i in range(n)]


def _flops(case):
    nq, _, d = HEADS[case["heads"]]
    if case["kind"] == "decode":
        return 4 * nq * d * sum(_lens(case["seqs"], case["ctx"]))
    if case["kind"] == "prompts":
        return 4 * nq * d * sum(n * case["ctx"] + n * (n + 1) // 2 for n in _lens(case["seqs"], case["len"]))
    return 6 * (nq + HEADS[case["heads"]][1]) * d // 2 * case["rows"]


def work(case):
    nq, nkv, d = HEADS[case["heads"]]
    row = 2 * nkv * (d // 2 + d // 32)                   # one token's K and V in 4 bits
    if case["kind"] in ("write", "axes"):
        T = case["rows"]
        n = T * (nq + 2 * nkv) * d * 2 + T * nq * d * 2 + T * 16 + min(T, 4096) * d * 4
        # the values read back
        n += T * (row + 2 * nkv * d * 2) if case.get("cache", "fp4") == "fp4" else T * 2 * nkv * d * 2
    elif case["kind"] == "decode":
        n = sum(_lens(case["seqs"], case["ctx"])) * row + 2 * case["seqs"] * nq * d * 2
    else:
        lens = _lens(case["seqs"], case["len"])
        n = sum(m + case["ctx"] for m in lens) * row + 2 * sum(lens) * nq * d * 2
    return {"bytes": n, "flops": _flops(case)}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _pages(g, tokens, nkv, d, dtype, spread):
    """A cache of ``tokens`` / PAGE pages of random rows, ``spread``: channels of unequal size."""
    nb = tokens // PAGE
    out = torch.empty(nb, nkv, PAGE, d // 2 + d // 32, dtype=torch.uint8, device="cuda")
    size = torch.exp(spread * torch.randn(nkv, 1, d, generator=g, device="cuda"))
    for at in range(0, nb, 4096):
        n = min(4096, nb - at)
        codes, e = _codes(torch.randn(n, nkv, PAGE, d, generator=g, device="cuda") * size, dtype)
        codes = codes.view(n, nkv, PAGE * d // 2, 2)
        out[at:at + n].view(n, nkv, -1)[..., :PAGE * d // 2] = codes[..., 0] | codes[..., 1] << 4
        out[at:at + n].view(n, nkv, -1)[..., PAGE * d // 2:] = (e + 127).to(torch.uint8).view(n, nkv, -1)
    return out


def _tables(g, totals):
    """Pages of every sequence, anywhere in the pool; page 0 is reserved."""
    width = -(-max(totals) // PAGE) + 1
    pages = len(totals) * width + 1
    tables = torch.randperm(pages - 1, generator=g, device="cuda") + 1
    return tables.view(len(totals), width).int(), pages


def _axis_positions(T):
    """Positions [3, T] of text, then frames of an image or video (each a grid of patches), then text:
    text turns all axes alike, a patch has its frame, row and column behind the text before it."""
    head = min(T, 17)
    side = max(1, int(math.sqrt(max(1, T // 3))) if T < 4000 else 32)
    n = max(0, T - head - 23)
    i = np.arange(n)
    grid = np.stack([i // (side * side), i // side % side, i % side]) + head
    p = np.concatenate([np.tile(np.arange(head), (3, 1)), grid], axis=1)
    tail = np.arange(T - p.shape[1]) + p.max() + 1
    return torch.from_numpy(np.concatenate([p, np.tile(tail, (3, 1))], axis=1).astype(np.int64))


def prepare(case, seed):
    g = _gen(seed)
    nq, nkv, d = HEADS[case["heads"]]
    dtype = DTYPES[case["dtype"]]
    s = dict(case=case, nq=nq, nkv=nkv, d=d, dtype=dtype, scale=d ** -0.5)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    if case["kind"] in ("write", "axes"):
        T = case["rows"]
        w = torch.exp(0.5 * torch.randn((nq + 2 * nkv) * d, generator=g, device="cuda"))
        s["qkv"] = (torch.randn(T, (nq + 2 * nkv) * d, generator=g, device="cuda") * w).to(dtype)
        if case["kind"] == "axes":
            s["positions"] = _axis_positions(T).cuda()
            s["sections"] = SECTIONS[d]
        elif T <= 256:
            s["positions"] = torch.randint(0, 8192, (T,), generator=g, device="cuda")
        else:                                             # prompts of 512
            s["positions"] = torch.arange(T, device="cuda") % 512
        inv = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
        a = (torch.arange(int(s["positions"].max()) + 1, dtype=torch.float64)[:, None] * inv).cuda()
        s["cos_sin"] = torch.cat([a.cos(), a.sin()], dim=1).float()
        pages = -(-T // PAGE) + 3
        order = torch.randperm(pages - 1, generator=g, device="cuda") + 1
        t = torch.arange(T, device="cuda")
        s["slots"] = order[t // PAGE] * PAGE + t % PAGE
        if case["pad"]:
            s["slots"][-case["pad"]:] = -1
        if case.get("cache", "fp4") == "fp4":
            s["k_cache"] = torch.zeros(pages, nkv, PAGE, d // 2 + d // 32, dtype=torch.uint8, device="cuda")
            s["v_cache"] = torch.zeros_like(s["k_cache"])
        else:
            s["k_cache"] = torch.zeros(pages, nkv, PAGE, d, dtype=dtype, device="cuda")
            s["v_cache"] = torch.zeros(pages, nkv, PAGE // 8, d, 8, dtype=dtype, device="cuda")
        return s
    if case["kind"] == "decode":
        totals = _lens(case["seqs"], case["ctx"])
        s["q"] = torch.randn(case["seqs"], nq, d, generator=g, device="cuda").to(dtype)
        s["ctx_lens"] = i32(totals)
    else:
        new = _lens(case["seqs"], case["len"])
        totals = [n + case["ctx"] for n in new]
        s["q"] = torch.randn(sum(new), nq, d, generator=g, device="cuda").to(dtype)
        s["starts"] = i32([0] + np.cumsum(new).tolist())
        s["seq_lens"] = i32(totals)
        # blocks of 128 query rows, those with most keys first
        items = sorted((-(case["ctx"] + min(128 * (m + 1), n)), i, m)
                       for i, n in enumerate(new) for m in range(-(-n // 128)))
        s["work"] = (i32([i for _, i, _ in items]), i32([m for _, _, m in items]))
        s["most_new"] = max(new)
    s["most"] = max(totals)
    s["tables"], pages = _tables(g, totals)
    s["k_cache"] = _pages(g, pages * PAGE, nkv, d, dtype, 0.5)
    s["v_cache"] = _pages(g, pages * PAGE, nkv, d, dtype, 0.2)
    return s


# ------------------------------------------------------------------ the plain forms
def _codes(x, dtype):
    """e2m1 codes of x and the exponents of its blocks of 32: the power of two under which the
    block's largest magnitude is at most 7 (what is over 6 is 6), ties to the even code."""
    b = x.unflatten(-1, (-1, 32))
    most = b.abs().amax(-1)
    m, e = torch.frexp(most)
    lo, hi = EXPONENTS[dtype]
    e = torch.where(most > 0, (e - 3 + (m > 0.875)).clamp(lo, hi), lo)
    a = torch.ldexp(b, -e.unsqueeze(-1)).abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5))
    return (code + 8 * (b < 0)).flatten(-2), e


def _values(codes, e):
    lut = torch.tensor(LUT + tuple(-v for v in LUT), device=codes.device)
    return torch.ldexp(lut[codes.long()].unflatten(-1, (-1, 32)), e.unsqueeze(-1)).flatten(-2)


def _widen(cache, pages, d):
    """The values of these pages [..., pages, kv heads, PAGE, d], fp32."""
    raw = cache.flatten(2)[pages.long()]
    n, sc = raw[..., :PAGE * d // 2], raw[..., PAGE * d // 2:]
    codes = torch.stack([n & 15, n >> 4], dim=-1).unflatten(-2, (PAGE, d // 2)).flatten(-2)
    return _values(codes, sc.int().unflatten(-1, (PAGE, d // 32)) - 127)


def _rotate(x, cos, sin):
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _write(s):
    nq, nkv, d, dtype, T = s["nq"], s["nkv"], s["d"], s["dtype"], s["qkv"].shape[0]
    q, k, v = s["qkv"].float().view(T, nq + 2 * nkv, d).split([nq, nkv, nkv], dim=1)
    if "sections" in s:
        axis = torch.repeat_interleave(torch.arange(3, device="cuda"), torch.tensor(s["sections"], device="cuda"),
                                       output_size=d // 2)
        at = s["positions"].t()[:, axis]                            # [T, d / 2]
    else:
        at = s["positions"][:, None].expand(T, d // 2)
    i = torch.arange(d // 2, device="cuda")
    cos, sin = s["cos_sin"][at, i][:, None], s["cos_sin"][at, i + d // 2][:, None]
    q = _rotate(q, cos, sin).to(dtype)
    there = (s["slots"] >= 0)[:, None, None]
    if s["k_cache"].dtype == torch.uint8:
        k = _rotate(k.double(), cos.double(), sin.double())     # next to a border of two codes
        return q, *(torch.where(there, _values(*_codes(x.contiguous(), dtype)), 0).to(dtype) for x in (k, v))
    k, v = _rotate(k, cos, sin).to(dtype), v.to(dtype)
    to = s["slots"].clamp(min=0)                                    # rows of no slot: page 0, as it was
    blk, off = to // PAGE, to % PAGE
    kc, vc = s["k_cache"].transpose(1, 2), s["v_cache"].permute(0, 2, 4, 1, 3)
    kc[blk, off] = torch.where(there, k, kc[0, 0])
    vc[blk, off // 8, off % 8] = torch.where(there, v, vc[0, 0, 0])
    return q, s["k_cache"], s["v_cache"]


def _attend(q, k, v, seen):
    """softmax(q k^T) v of q [n, kv heads, rows, d]; ``seen`` [n, 1, rows or 1, keys]."""
    p = q @ k.transpose(2, 3)
    p = p.masked_fill_(~seen, -math.inf)
    m = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(m > -math.inf, m, 0)).exp_()
    total = p.sum(-1, keepdim=True)
    return p @ v / torch.where(total > 0, total, 1)


def _decode(s):
    nq, nkv, d = s["nq"], s["nkv"], s["d"]
    B = s["q"].shape[0]
    k, v = (_widen(c, s["tables"], d).transpose(1, 2).flatten(2, 3) for c in (s["k_cache"], s["v_cache"]))
    seen = torch.arange(k.shape[2], device="cuda") < s["ctx_lens"][:, None]
    q = s["q"].float().view(B, nkv, nq // nkv, d) * s["scale"]
    return _attend(q, k, v, seen[:, None, None]).view(B, nq, d).to(s["dtype"])


def _prompts(s):
    nq, nkv, d = s["nq"], s["nkv"], s["d"]
    k, v = (_widen(c, s["tables"], d).transpose(1, 2).flatten(2, 3) for c in (s["k_cache"], s["v_cache"]))
    P, most, T = k.shape[0], s["most_new"], s["q"].shape[0]
    begin, new = s["starts"][:-1].long(), (s["starts"][1:] - s["starts"][:-1]).long()
    r = torch.arange(most, device="cuda")
    q = s["q"][(begin[:, None] + r).clamp(max=T - 1)]                # [P, most, nq, d]
    q = q.float().view(P, most, nkv, nq // nkv, d).permute(0, 2, 3, 1, 4).flatten(2, 3) * s["scale"]
    last = (s["seq_lens"] - new)[:, None] + r                       # the row's own position
    seen = torch.arange(k.shape[2], device="cuda") <= last[..., None]
    o = _attend(q, k, v, seen.repeat(1, nq // nkv, 1)[:, None])
    o = o.view(P, nkv, nq // nkv, most, d).permute(0, 3, 1, 2, 4).flatten(2, 3)
    t = torch.arange(T, device="cuda")
    i = torch.searchsorted(s["starts"][1:].long(), t, right=True)
    return o[i, t - begin[i]].to(s["dtype"])


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return _write(s) if kind in ("write", "axes") else _decode(s) if kind == "decode" else _prompts(s)
    from kubernetes_gpu_cluster_amd import ops
    kc, vc = s["k_cache"], s["v_cache"]
    if kind in ("write", "axes"):
        q = ops.rope_kv_write(s["qkv"], s["positions"], s["cos_sin"], kc, vc, s["slots"], s["nq"], s["nkv"],
                              s["d"], sections=s.get("sections"))
        if kc.dtype != torch.uint8:
            return q, kc, vc
        return q, ops.kv4_read(kc, s["slots"], s["dtype"]), ops.kv4_read(vc, s["slots"], s["dtype"])
    if kind == "decode":
        B, nq, d = s["q"].shape
        if "partials" not in s:                            # a program's own: once
            s["partials"] = ops.decode_partials(B, nq, d, s["tables"].shape[1], PAGE, s["q"].device)
        z = ops.decode_grid_z(B, s["nkv"], s["most"], cache_dtype=kc.dtype)
        return ops.paged_attention_decode(s["q"], kc, vc, s["tables"], s["ctx_lens"], s["scale"], s["partials"], z)
    return ops.prefill_attention(s["q"], kc, vc, s["tables"], s["starts"], s["seq_lens"], s["scale"], *s["work"],
                                 max_len=s["most"])


# ------------------------------------------------------------------ 64 bits
_E2M1 = torch.tensor([(-1.0 if c & 8 else 1.0) * ((c & 1) * 0.5 if not c & 6 else (1 + (c & 1) / 2) * 2.0 ** ((c >> 1 & 3) - 1))
                      for c in range(16)], dtype=torch.float64)


def _page_rows(cache, pages, h, n, d):
    """The first n rows of kv head h in these pages, 64 bits."""
    flat = cache[pages.long(), h].reshape(len(pages), -1).long()
    at = torch.arange(PAGE * d, device=cache.device)
    code = flat[:, at // 2] >> 4 * (at % 2) & 15
    size = torch.pow(2.0, (flat[:, PAGE * d // 2 + at // 32] - 127).double())
    return (_E2M1.to(cache.device)[code] * size).view(-1, d)[:n]


def _nearest(x, dtype):
    """The values that a 4-bit cache holds for x [..., d], 64 bits: by distance to every code."""
    b = x.reshape(-1, 32)
    most = b.abs().max(dim=1).values
    e = torch.floor(torch.log2(most.clamp(min=1e-300)))
    e = e + (most >= torch.pow(2.0, e + 1)).double() - (most < torch.pow(2.0, e)).double()
    e = (e - 2 + (most > 1.75 * torch.pow(2.0, e)).double()).clamp(*EXPONENTS[dtype])
    size = torch.pow(2.0, e)[:, None]
    table = _E2M1[:8].to(x.device)
    a = (b / size).abs()
    best, far = torch.zeros_like(a), torch.full_like(a, math.inf)
    for c in (0, 2, 4, 6, 1, 3, 5, 7):                    # the even codes first: they keep a tie
        off = (a - table[c]).abs()
        best, far = torch.where(off < far, table[c], best), torch.minimum(off, far)
    return (best * b.sign() * size).view(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    nq, nkv, d = s["nq"], s["nkv"], s["d"]
    if case["kind"] in ("write", "axes"):
        T = case["rows"]
        x = s["qkv"].double().view(T, nq + 2 * nkv, d)
        turned = torch.empty(T, nq + nkv, d, dtype=torch.float64, device=x.device)
        axis = [a for a, n in enumerate(s["sections"]) for _ in range(n)] if "sections" in s else None
        for i in range(d // 2):
            p = s["positions"] if axis is None else s["positions"][axis[i]]
            c, n = s["cos_sin"][p, i].double()[:, None], s["cos_sin"][p, d // 2 + i].double()[:, None]
            a, b = x[:, :nq + nkv, i], x[:, :nq + nkv, d // 2 + i]
            turned[:, :, i], turned[:, :, d // 2 + i] = a * c - b * n, a * n + b * c
        k, v, slots = turned[:, nq:], x[:, nq + nkv:], s["slots"]
        if case.get("cache", "fp4") == "fp4":
            gone = slots < 0
            k, v = _nearest(k.contiguous(), s["dtype"]), _nearest(v.contiguous(), s["dtype"])
            k[gone], v[gone] = 0, 0
            return turned[:, :nq], k, v
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        t = torch.nonzero(slots >= 0)[:, 0]
        for h in range(nkv):
            kc[slots[t] // PAGE, h, slots[t] % PAGE] = k[t, h]
            for j in range(8):
                u = t[slots[t] % 8 == j]
                vc[slots[u] // PAGE, h, slots[u] % PAGE // 8, :, j] = v[u, h]
        return turned[:, :nq], kc, vc
    decode = case["kind"] == "decode"
    totals = (s["ctx_lens"] if decode else s["seq_lens"]).tolist()
    starts = list(range(len(totals) + 1)) if decode else s["starts"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(totals):
        if not n:
            continue
        rows = slice(starts[i], starts[i + 1])
        m = starts[i + 1] - starts[i]
        pages = s["tables"][i, :-(-n // PAGE)]
        hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - m, n, device="cuda")[:, None]
        for h in range(nkv):
            k, v = (_page_rows(c, pages, h, n, d) for c in (s["k_cache"], s["v_cache"]))
            for j in range(h * (nq // nkv), (h + 1) * (nq // nkv)):
                p = torch.softmax((s["q"][rows, j].double() @ k.T * d ** -0.5).masked_fill(hidden, -math.inf), dim=-1)
                out[rows, j] = p @ v
    return out
