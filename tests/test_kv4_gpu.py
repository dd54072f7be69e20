"""The 4-bit cache's kernels (csrc/kernels/kv4_*.hip) and rotary positions on several axes against 64 bits."""
import math

import pytest
import torch

import kv4_oracle as oracle
from kubernetes_gpu_cluster_amd import ops
from kubernetes_gpu_cluster_amd.ops import reference as ref

pytestmark = pytest.mark.gpu

DT = [torch.bfloat16, torch.float16]


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def _check_rows(got, want, u, size):
    """fp32 products and sum of two terms of at most ``size`` (3 roundings each 2^-24 relative of 2 size), then
    one rounding to the type (or its smallest step, fp16's 2^-25)."""
    tol = u * 1.01 * want.abs() + 6 * 2.0 ** -24 * size + 2.0 ** -25
    assert ((got.double() - want).abs() <= tol).all()


# ------------------------------------------------------------------ write
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("nq,nkv,d,bs", [(32, 8, 128, 32), (5, 1, 64, 16), (3, 3, 128, 64), (12, 12, 64, 32)])
@pytest.mark.parametrize("T,sections,slices", [(1, None, 0), (133, None, 0), (133, (10, 9, -1), 0), (37, None, 3),
                                               (37, (8, 8, 8, -1), 2), (300, (-1,), 0), (1500, (9, -1), 0)])
def test_write(gpu, dt, nq, nkv, d, bs, T, sections, slices):
    g = _gen(T + d)
    if sections:
        sections = [n if n >= 0 else d // 2 - sum(n for n in sections if n >= 0) for n in sections]
    nb = -(-T // bs) + 2
    kc = oracle.random_cache(g, nb, nkv, bs, d, dt)
    vc = oracle.random_cache(g, nb, nkv, bs, d, dt)
    width = (nq + 2 * nkv) * d
    x = torch.randn(max(slices, 1), T, width, generator=g) * torch.exp(torch.randn(width, generator=g))
    qkv = x.float() if slices else torch.cat([x[0].to(dt), torch.zeros(T, 16, dtype=dt)], 1)   # rows of a wider matrix
    slots = torch.randperm(nb * bs, generator=g)[:T]
    if T > 30:
        slots[7], slots[T - 1] = -1, nb * bs + 5              # graph padding; beyond the pool
    table = ref.rope_cos_sin_cache(d, 400, 10000.0)
    pos = torch.randint(0, 400, (len(sections), T) if sections else (T,), generator=g)
    kg, vg = kc.to(gpu), vc.to(gpu)
    q = ops.rope_kv_write(qkv.to(gpu), pos.to(gpu), table.to(gpu), kg, vg, slots.to(gpu), nq, nkv, d, dtype=dt,
                          sections=sections)
    # slices are summed in fp32, in order, and rounded to the type
    rows = qkv[:, :width] if not slices else x[0]
    for z in range(1, slices):
        rows = rows + x[z]
    rows = rows.to(dt).view(T, nq + 2 * nkv, d).double()
    cos, sin = oracle.cos_sin_rows(table, pos, sections)
    _check_rows(q.cpu(), oracle.rotate(rows[:, :nq], cos, sin), torch.finfo(dt).eps / 2, 2 * rows.abs().max())
    k = oracle.nearest(oracle.rotate(rows[:, nq:nq + nkv], cos, sin), dt)[0]
    v = oracle.nearest(rows[:, nq + nkv:], dt)[0]
    there = (slots >= 0) & (slots < nb * bs)
    for got, want, old in ((kg, k, kc), (vg, v, vc)):
        back = ops.kv4_read(got, slots.to(gpu), dt).cpu()
        assert torch.equal(back[there].double(), want[there]) and not back[~there].any()
        for part, was in zip(ref.kv4_parts(got.cpu()), ref.kv4_parts(old)):      # all other bytes as they were
            part, was = part.transpose(1, 2).flatten(0, 1), was.transpose(1, 2).flatten(0, 1)
            kept = torch.ones(nb * bs, dtype=torch.bool)
            kept[slots[there]] = False
            assert torch.equal(part[kept], was[kept])
        n, s = (p[slots[there] // bs, :, slots[there] % bs] for p in ref.kv4_parts(got.cpu()))
        assert torch.equal(ref.kv4_dequantize(n, s).double(), want[there])


@pytest.mark.parametrize("dt", DT)
def test_write_unrotated_and_special(gpu, dt):
    """Ties, the scales' ends, subnormal blocks, zeros, infinities and NaN."""
    d, T = 64, 9
    x = torch.randn(T, 3, d, generator=_gen(5))
    x[0, :, :32] = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6] * 4)
    x[1] = -x[0] * 2.0 ** -7
    x[2, :, 0], x[2, :, 32] = 60000.0, 7.0
    x[3], x[4] = x[3] * 2.0 ** -20, 0
    x[5, :, 1] = float("inf")
    x[6, :, 2], x[6, :, 3] = float("nan"), -float("inf")
    x[7, :, 0] = 7.0625
    x = x.to(dt)
    kc, vc = (torch.zeros(ops.kv4_cache_shape(2, 1, 16, d), dtype=torch.uint8, device=gpu) for _ in range(2))
    slots = torch.arange(T, device=gpu)
    table = ref.rope_cos_sin_cache(d, 4, 10000.0).to(gpu)
    q = ops.rope_kv_write(x.view(T, -1).to(gpu), slots * 0, table, kc, vc, slots, 1, 1, d, use_rope=False)
    assert torch.equal(q.cpu().nan_to_num(7), x[:, :1].nan_to_num(7))
    for c, want in ((kc, x[:, 1:2]), (vc, x[:, 2:])):
        n, s = ref.kv4_quantize(want, dt)
        for got, w in zip(ref.kv4_parts(c.cpu()), (n, s)):
            got = got[0, :, :T].transpose(0, 1)
            if w is n:                                       # (a zero's sign is not kept by all)
                got, w = ref.kv4_dequantize(got, s), ref.kv4_dequantize(w, s)
            assert torch.equal(got, w)
        assert ops.kv4_read(c, slots, dt).isfinite().all()


@pytest.mark.parametrize("cache", ["fp4", "auto"])
@pytest.mark.parametrize("sections", [None, (24, 20, 20)])
def test_write_with_norms(gpu, cache, sections):
    """q / k norms: k's codes are within the step of what 64 bits give, for the norm's rounding to the type."""
    g, dt, nq, nkv, d, T = _gen(6), torch.bfloat16, 8, 2, 128, 50
    x = torch.randn(T, (nq + 2 * nkv) * d, generator=g).to(dt)
    qw, kw = (torch.rand(d, generator=g).add(0.5).to(dt) for _ in range(2))
    table = ref.rope_cos_sin_cache(d, 100, 10000.0)
    pos = torch.randint(0, 100, (3, T) if sections else (T,), generator=g)
    shape = ops.kv4_cache_shape(2, nkv, 32, d)
    kc, vc = ((torch.zeros(shape, dtype=torch.uint8, device=gpu) for _ in range(2)) if cache == "fp4" else
              (torch.zeros(2, nkv, 32, d, dtype=dt, device=gpu), torch.zeros(2, nkv, 4, d, 8, dtype=dt, device=gpu)))
    slots = torch.randperm(64, generator=g)[:T]
    q = ops.rope_kv_write(x.to(gpu), pos.to(gpu), table.to(gpu), kc, vc, slots.to(gpu), nq, nkv, d, qw.to(gpu),
                          kw.to(gpu), 1e-6, sections=sections)
    h = x.double().view(T, -1, d)
    h = h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    cos, sin = oracle.cos_sin_rows(table, pos, sections)
    # the norm's result is rounded to the type (2^-8 of each of the two terms) before the rotation
    qn, kn = h[:, :nq] * qw.double(), h[:, nq:nq + nkv] * kw.double()
    off = lambda y: (1.01 * 2.0 ** -8 + 2.0 ** -20) * oracle.rotate(y.abs(), cos.abs(), -sin.abs()).abs() + \
        (1.01 * 2.0 ** -8 + 2.0 ** -20) * oracle.rotate(y.abs(), cos.abs(), sin.abs()).abs()    # noqa: E731
    want = oracle.rotate(qn, cos, sin)
    assert ((q.cpu().double() - want).abs() <= off(qn) + 1.01 * 2.0 ** -8 * (want.abs() + off(qn))).all()
    want = oracle.rotate(kn, cos, sin)
    if cache == "fp4":
        got = ops.kv4_read(kc, slots.to(gpu), dt).cpu().double()
        e = ref.kv4_parts(kc.cpu())[1][slots // 32, :, slots % 32].double() - 127
        step = (2 ** e).repeat_interleave(32, -1)            # no number is further than this from its code
    else:
        got, step = kc.cpu().double()[slots // 32, :, slots % 32], 1.01 * 2.0 ** -8 * (want.abs() + off(kn))
    assert ((got - want).abs() <= step + off(kn)).all()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("cache", ["auto", "fp8"])
@pytest.mark.parametrize("T,sections,slices", [(77, (16, 24, 24), 0), (77, (5, 0, 40, 19), 0), (9, (64,), 2), (700, (16, 24, 24), 0),
                                               (521, (60, 1, 3), 0), (2851, (16, 24, 24), 0), (2400, (3, 50, 11), 0)])
def test_axes_of_the_wider_caches(gpu, dt, cache, T, sections, slices):
    g, nq, nkv, d, bs = _gen(7), 8, 2, 128, 16
    t = torch.float8_e4m3fn if cache == "fp8" else dt
    nb = max(8, T // 16 + 3)
    mk = lambda: (torch.zeros(nb, nkv, bs, d).to(t).to(gpu), torch.zeros(nb, nkv, bs // 8, d, 8).to(t).to(gpu))   # noqa: E731
    x = torch.randn(max(slices, 1), T, (nq + 2 * nkv) * d, generator=g)
    x = x.to(gpu) if slices else x[0].to(dt).to(gpu)
    table = ref.rope_cos_sin_cache(d, 90, 10000.0)
    pos = torch.randint(-5, 99, (len(sections), T), generator=g)
    slots = torch.randperm(nb * bs, generator=g)[:T]
    if T > 100:                                               # runs that start in an 8-key group, and padding
        slots = (torch.arange(T) + 5) % (nb * bs)
        slots[100:] += 3
        slots[-3:] = -1
    slots = slots.to(gpu)
    kc, vc = mk()
    q = ops.rope_kv_write(x, pos.to(gpu), table.to(gpu), kc, vc, slots, nq, nkv, d, dtype=dt, sections=sections)
    # each pair as the one-position kernel turns it, from a table of that axis's rows
    for a, n in enumerate(sections):
        rows = table[pos[a].clamp(0, 89)].contiguous().to(gpu)
        k2, v2 = mk()
        q2 = ops.rope_kv_write(x, torch.arange(T, device=gpu), rows, k2, v2, slots, nq, nkv, d, dtype=dt)
        i = torch.arange(sum(sections[:a]), sum(sections[:a + 1]), device=gpu)
        i = torch.cat([i, i + d // 2])
        assert torch.equal(q[..., i], q2[..., i])
        assert torch.equal(kc.float()[..., i], k2.float()[..., i]) and torch.equal(vc.float(), v2.float())


# ------------------------------------------------------------------ attention
def _attention_case(seed, nq, nkv, d, bs, dt, new, old, k_size=1.0):
    g = _gen(seed)
    totals = [a + b for a, b in zip(new, old)]
    bt, nb = oracle.tables(g, totals, bs)
    kc = oracle.random_cache(g, nb, nkv, bs, d, dt, k_size)
    vc = oracle.random_cache(g, nb, nkv, bs, d, dt)
    kc[0], vc[0] = 255, 255                                   # nobody's page: no finite value
    for c in (kc, vc):                                        # and behind the last tokens
        for i, n in enumerate(totals):
            if n % bs:
                for p in ref.kv4_parts(c):
                    p[bt[i, n // bs], :, n % bs:] = 255
    q = torch.randn(sum(new), nq, d, generator=g).to(dt)
    return q, kc, vc, bt, totals


def _check_attention(got, q, kc, vc, bt, new, totals, scale):
    nq, nkv, d = q.shape[1], kc.shape[1], q.shape[2]
    at = 0
    for i, (m, n) in enumerate(zip(new, totals)):
        if n == 0:
            assert not got[at:at + m].any()
            at += m
            continue
        seen = torch.arange(n)[None] <= torch.arange(n - m, n)[:, None]
        for h in range(nkv):
            k, v = (oracle.rows(c, bt[i], n, h, d) for c in (kc, vc))
            for j in range(h * (nq // nkv), (h + 1) * (nq // nkv)):
                o, tol = oracle.attend(q[at:at + m, j], k, v, scale, seen, q.dtype)
                off = (got[at:at + m, j].double() - o).abs()
                assert (off <= tol).all(), (i, j, float((off / tol).max()))
        at += m


DECODE = [
    # q heads, kv heads, head, page, contexts
    (4, 1, 128, 32, [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100]),
    (32, 8, 128, 32, [640, 1, 0, 333]),
    (12, 12, 64, 16, [47, 200, 1]),
    (16, 1, 64, 64, [129, 5]),
    (8, 8, 128, 16, [1500]),
    (10, 2, 64, 32, [500, 31, 96]),
    (7, 1, 128, 128, [257, 128]),
    (8, 8, 64, 32, [2100, 1, 0, 90, 64, 33, 500, 2, 7]),
    (8, 8, 64, 16, [1 + 7 * i % 67 for i in range(70)]),
    (8, 8, 64, 32, [3 * i % 71 for i in range(130)]),
    (4, 4, 64, 32, [5 * i % 77 for i in range(400)]),
]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("nq,nkv,d,bs,ctx", DECODE)
@pytest.mark.parametrize("z", [1, 2, 3, 0, 64])
def test_decode(gpu, dt, nq, nkv, d, bs, ctx, z):
    q, kc, vc, bt, _ = _attention_case(sum(ctx), nq, nkv, d, bs, dt, [1] * len(ctx), [c - 1 for c in ctx])
    ws = ops.decode_partials(len(ctx), nq, d, 64 * 64 // bs, bs, gpu)
    for t in ws:
        t.fill_(float("nan"))                                 # no slice is read that none wrote
    z = z or ops.decode_grid_z(len(ctx), nkv, max(ctx), cache_dtype=torch.uint8)
    out = torch.full_like(q, 7).to(gpu)
    got = ops.paged_attention_decode(q.to(gpu), kc.to(gpu), vc.to(gpu), bt.to(gpu),
                                     torch.tensor(ctx, dtype=torch.int32, device=gpu), d ** -0.5, ws, z, out=out)
    assert got.data_ptr() == out.data_ptr()
    _check_attention(got.cpu(), q, kc, vc, bt, [1] * len(ctx), ctx, d ** -0.5)
    own = ops.paged_attention_decode(q.to(gpu), kc.to(gpu), vc.to(gpu), bt.to(gpu),
                                     torch.tensor(ctx, dtype=torch.int32, device=gpu), d ** -0.5, None, z)
    assert torch.equal(own, got)


@pytest.mark.parametrize("dt", DT)
def test_decode_sharp_rows(gpu, dt):
    """Keys large enough that one token has all the weight, and scores far apart between slices."""
    ctx = [700, 90, 33]
    q, kc, vc, bt, _ = _attention_case(3, 8, 2, 128, 32, dt, [1] * 3, [c - 1 for c in ctx], k_size=32.0)
    for z in (1, 4, 11):
        got = ops.paged_attention_decode(q.to(gpu), kc.to(gpu), vc.to(gpu), bt.to(gpu),
                                         torch.tensor(ctx, dtype=torch.int32, device=gpu), 0.25, None, z)
        _check_attention(got.cpu(), q, kc, vc, bt, [1] * 3, ctx, 0.25)


PROMPTS = [
    # q heads, kv heads, head, page, new rows, cached before
    (4, 1, 128, 32, [1, 2, 31, 32, 33, 64, 65], [0, 0, 0, 0, 0, 0, 0]),
    (32, 8, 128, 32, [130, 1, 257], [0, 63, 100]),
    (12, 12, 64, 16, [128, 3, 47], [16, 15, 17]),
    (2, 1, 128, 64, [200], [5]),
    (6, 2, 64, 32, [129, 64], [700, 0]),
    (16, 1, 128, 16, [33, 90], [31, 1]),
    (7, 1, 64, 32, [300], [0]),
    (1, 1, 128, 32, [1, 1, 1], [0, 64, 255]),
    # many items
    (32, 8, 128, 32, [1 + 17 * i % 150 for i in range(60)], [5 * i % 90 for i in range(60)]),
    (12, 12, 64, 16, [2 + 11 * i % 130 for i in range(100)], [7 * i % 40 for i in range(100)]),
    (12, 6, 128, 64, [3 + 29 * i % 140 for i in range(70)], [0] * 70),
]


def _starts(new):
    return torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("nq,nkv,d,bs,new,old", PROMPTS)
def test_prompts(gpu, dt, nq, nkv, d, bs, new, old):
    q, kc, vc, bt, totals = _attention_case(sum(new), nq, nkv, d, bs, dt, new, old)
    qg = torch.cat([q, torch.zeros(3, nq, d, dtype=dt)]).to(gpu)
    out = torch.full_like(qg, 7)                              # rows behind the last sequence: as they were
    got = ops.prefill_attention(qg, kc.to(gpu), vc.to(gpu), bt.to(gpu), _starts(new).to(gpu),
                                torch.tensor(totals, dtype=torch.int32, device=gpu), d ** -0.5, out=out)
    assert got.data_ptr() == out.data_ptr() and (out[-3:] == 7).all()
    _check_attention(got[:-3].cpu(), q, kc, vc, bt, new, totals, d ** -0.5)
    own = ops.prefill_attention(q.to(gpu), kc.to(gpu), vc.to(gpu), bt.to(gpu), _starts(new).to(gpu),
                                torch.tensor(totals, dtype=torch.int32, device=gpu), d ** -0.5)
    _check_attention(own.cpu(), q, kc, vc, bt, new, totals, d ** -0.5)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("nq,nkv,d,bs,new,old", [
    (4, 1, 128, 32, [33, 1, 130], [1900, 700, 0]),
    (3, 3, 64, 16, [40, 5], [0, 1000]),
    (16, 2, 128, 64, [7], [1500]),
])
@pytest.mark.parametrize("z", [2, 5, 32])
def test_prompts_in_slices(gpu, dt, nq, nkv, d, bs, new, old, z):
    """z workgroups per item, among them some that see nothing; the merge leaves other rows as they were."""
    q, kc, vc, bt, totals = _attention_case(z + sum(new), nq, nkv, d, bs, dt, new, old)
    qg = torch.cat([q, torch.zeros(3, nq, d, dtype=dt)]).to(gpu)
    ws, wm = (torch.tensor(w, dtype=torch.int32, device=gpu) for w in ops.prefill_work_list(new, totals))
    parts = torch.full((z * len(qg) * nq * (d + 2),), float("nan"), device=gpu)
    out = torch.full_like(qg, 7)
    torch.ops.kgc.prefill_attention(out, qg, kc.to(gpu), vc.to(gpu), bt.to(gpu), _starts(new).to(gpu),
                                    torch.tensor(totals, dtype=torch.int32, device=gpu), ws, wm, d ** -0.5, 1.0, 1.0, 0,
                                    parts)
    assert (out[-3:] == 7).all()
    _check_attention(out[:-3].cpu(), q, kc, vc, bt, new, totals, d ** -0.5)


@pytest.mark.parametrize("z", [1, 3])
def test_nan_queries_stay_with_their_rows(gpu, z):
    """A NaN or infinite query row is NaN, with slices too, and no other row is."""
    new, old = [70, 3], [600, 900]
    q, kc, vc, bt, totals = _attention_case(2, 4, 2, 64, 32, torch.bfloat16, new, old)
    q[5, 1], q[71, 2, 7] = float("nan"), float("inf")
    n = torch.tensor(totals, dtype=torch.int32, device=gpu)
    ws, wm = (torch.tensor(w, dtype=torch.int32, device=gpu) for w in ops.prefill_work_list(new, totals))
    parts = torch.empty(z * q.numel() // 64 * 66, device=gpu) if z > 1 else None
    out = torch.empty_like(q).to(gpu)
    torch.ops.kgc.prefill_attention(out, q.to(gpu), kc.to(gpu), vc.to(gpu), bt.to(gpu), _starts(new).to(gpu), n, ws, wm,
                                    0.125, 1.0, 1.0, 0, parts)
    bad = torch.zeros(73, 4, dtype=torch.bool)
    bad[5, 1] = bad[71, 2] = True
    assert torch.equal(out.cpu().isnan().all(-1), bad) and torch.equal(out.cpu().isnan().any(-1), bad)
    dec = ops.paged_attention_decode(q[4:6].contiguous().to(gpu), kc.to(gpu), vc.to(gpu), bt.to(gpu), n, 0.125, None, z)
    assert torch.equal(dec.cpu().isnan().all(-1), bad[4:6]) and torch.equal(dec.cpu().isnan().any(-1), bad[4:6])


def test_tables_and_lists_out_of_range(gpu):
    """Page numbers, lengths and work items that are none: other rows are right, and nothing is read or written
    elsewhere (the kernels clamp pages and lengths to the pool and leave such items out)."""
    if ops.DEBUG:
        pytest.skip("the bounds-checking build reports them")
    new, old = [20, 40], [100, 300]
    q, kc, vc, bt, totals = _attention_case(9, 4, 2, 64, 32, torch.bfloat16, new, old)
    bad = bt.clone()
    bad[0, 0], bad[0, 2] = -7, 1 << 30
    a = [t.to(gpu) for t in (kc, vc, bad)]
    n = torch.tensor(totals, dtype=torch.int32, device=gpu)
    last = torch.stack([q[19], q[59], q[0]]).to(gpu)
    bt3 = torch.cat([a[2], a[2][1:]])
    dec = ops.paged_attention_decode(last, a[0], a[1], bt3, torch.tensor([120, 340, -5], dtype=torch.int32, device=gpu),
                                     0.125, None, 2)
    assert not dec[2].any()
    _check_attention(dec[1:2].cpu(), q[59:], kc, vc, bt[1:], [1], totals[1:], 0.125)
    ws = torch.tensor([1, 7, -1, 0, 1], dtype=torch.int32, device=gpu)
    wm = torch.tensor([0, 0, 0, -1, 5], dtype=torch.int32, device=gpu)
    for z in (1, 4):
        out = torch.full_like(q, 7).to(gpu)
        torch.ops.kgc.prefill_attention(out, q.to(gpu), *a, _starts(new).to(gpu), n, ws, wm, 0.125, 1.0, 1.0, 0,
                                        torch.empty(z * q.numel() // 64 * 66, device=gpu))
        assert (out[:20] == 7).all()
        _check_attention(out[20:].cpu(), q[20:], kc, vc, bt[1:], new[1:], totals[1:], 0.125)
        starts = torch.tensor([-3, 0, 999], dtype=torch.int32, device=gpu)
        out.fill_(7)
        torch.ops.kgc.prefill_attention(out, q.to(gpu), *a, starts, n, ws, wm, 0.125, 1.0, 1.0, 0,
                                        torch.empty(z * q.numel() // 64 * 66, device=gpu))
        assert (out == 7).all()


@pytest.mark.parametrize("dt", DT)
def test_prompts_sharp_rows(gpu, dt):
    new, old = [150, 40], [90, 0]
    q, kc, vc, bt, totals = _attention_case(11, 8, 2, 128, 32, dt, new, old, k_size=32.0)
    got = ops.prefill_attention(q.to(gpu), kc.to(gpu), vc.to(gpu), bt.to(gpu), _starts(new).to(gpu),
                                torch.tensor(totals, dtype=torch.int32, device=gpu), 0.25)
    _check_attention(got.cpu(), q, kc, vc, bt, new, totals, 0.25)


def test_empty_calls(gpu):
    kc = torch.zeros(ops.kv4_cache_shape(3, 2, 16, 64), dtype=torch.uint8, device=gpu)
    i32 = lambda *n: torch.zeros(*n, dtype=torch.int32, device=gpu)   # noqa: E731
    q = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=gpu)
    assert ops.paged_attention_decode(q, kc, kc, i32(0, 2), i32(0), 1.0).shape == q.shape
    assert ops.prefill_attention(q, kc, kc, i32(1, 2), i32(2), i32(1), 1.0).shape == q.shape
    table = torch.zeros(4, 64, device=gpu)
    none = torch.zeros(0, dtype=torch.int64, device=gpu)
    assert ops.rope_kv_write(torch.zeros(0, 512, dtype=torch.bfloat16, device=gpu), none, table, kc, kc.clone(), none,
                             4, 2, 64).shape == q.shape
    assert ops.kv4_read(kc, none, torch.float16).shape == (0, 2, 64)


# ------------------------------------------------------------------ together
def _prompt_then_decode(dev, dt, graph):
    """A prompt in two chunks, then decode steps, as the engine calls the operators; positions on three axes.
    -> attention results, on the CPU."""
    g, nq, nkv, d, bs, n = _gen(21), 8, 2, 128, 32, 75
    shape = ops.kv4_cache_shape(5, nkv, bs, d)
    kc, vc = (torch.zeros(shape, dtype=torch.uint8, device=dev) for _ in range(2))
    table = ref.rope_cos_sin_cache(d, 128, 10000.0).to(dev)
    bt = torch.tensor([[3, 1, 4, 0]], dtype=torch.int32, device=dev)
    x = torch.randn(n + 6, (nq + 2 * nkv) * d, generator=g).to(dt).to(dev)
    pos = torch.stack([torch.arange(n + 6), torch.arange(n + 6) // 2, torch.arange(n + 6) % 7]).to(dev)
    slots = (bt[0].long()[torch.arange(n + 6, device=dev) // bs] * bs + torch.arange(n + 6, device=dev) % bs)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)   # noqa: E731
    sec, out = (16, 24, 24), []
    for a, b in ((0, 40), (40, n)):
        q = ops.rope_kv_write(x[a:b], pos[:, a:b], table, kc, vc, slots[a:b], nq, nkv, d, sections=sec)
        out.append(ops.prefill_attention(q, kc, vc, bt, i32(0, b - a), i32(b), d ** -0.5))
    ws = ops.decode_partials(1, nq, d, 4, bs, dev) if graph else None
    row, at, slot, length = x[:1].clone(), pos[:, :1].clone(), slots[:1].clone(), i32(0)

    def step():
        q = ops.rope_kv_write(row, at, table, kc, vc, slot, nq, nkv, d, sections=sec)
        return ops.paged_attention_decode(q, kc, vc, bt, length, d ** -0.5, ws, 2)
    run = None
    for t in range(n, n + 6):
        row.copy_(x[t:t + 1]), at.copy_(pos[:, t:t + 1]), slot.copy_(slots[t:t + 1]), length.fill_(t + 1)
        if graph and run is None:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            run = torch.cuda.CUDAGraph()
            with torch.cuda.graph(run):
                held = step()
        if graph:
            run.replay()
            out.append(held.clone())
            torch.cuda.synchronize()
        else:
            out.append(step())
    return [o.cpu() for o in out], kc.cpu(), vc.cpu()


@pytest.mark.parametrize("dt", DT)
def test_prompt_then_decode(gpu, dt):
    """The same run eagerly, with decode steps as replays of one captured graph, and on the CPU: equal caches; and
    results, to the type's rounding, of the CPU's."""
    eager, kc, vc = _prompt_then_decode(gpu, dt, False)
    graph, kc2, vc2 = _prompt_then_decode(gpu, dt, True)
    cpu, kc3, vc3 = _prompt_then_decode(torch.device("cpu"), dt, False)
    assert torch.equal(kc, kc2) and torch.equal(vc, vc2)
    for a, b in ((kc, kc3), (vc, vc3)):
        (n, s), (m, r) = ref.kv4_parts(a), ref.kv4_parts(b)
        used = [3, 1, 4]
        assert torch.equal(ref.kv4_dequantize(n[used], s[used]), ref.kv4_dequantize(m[used], r[used]))
    for a, b, c in zip(eager, graph, cpu):
        assert torch.equal(a, b)
        # two roundings of probabilities' products and results on one side, one on the other, of values below 8
        assert ((a.double() - c.double()).abs() <= 3 * torch.finfo(dt).eps * 8).all()


def test_pool_beyond_32_bits(gpu):
    """Pages behind the first 4 GB of a pool: written, read back and attended as in a small one."""
    g, dt, nq, nkv, d, bs, n = _gen(31), torch.bfloat16, 4, 1, 128, 32, 130
    nb = (9 << 29) // (bs * ref.kv4_row_bytes(d))             # 4.8 GB each
    big = [torch.zeros(ops.kv4_cache_shape(nb, nkv, bs, d), dtype=torch.uint8, device=gpu) for _ in range(2)]
    small = [torch.zeros(ops.kv4_cache_shape(6, nkv, bs, d), dtype=torch.uint8, device=gpu) for _ in range(2)]
    x = torch.randn(n, (nq + 2 * nkv) * d, generator=g).to(dt).to(gpu)
    pos = torch.arange(n, device=gpu)
    table = ref.rope_cos_sin_cache(d, 200, 10000.0).to(gpu)
    got = []
    for (kc, vc), first in ((big, nb - 5), (small, 1)):
        slots = pos + first * bs
        q = ops.rope_kv_write(x, pos, table, kc, vc, slots, nq, nkv, d)
        bt = torch.arange(first, first + 5, dtype=torch.int32, device=gpu)[None]
        ctx = torch.tensor([n], dtype=torch.int32, device=gpu)
        starts = torch.tensor([0, n], dtype=torch.int32, device=gpu)
        got.append([q, ops.kv4_read(kc, slots, dt), ops.kv4_read(vc, slots, dt),
                    ops.prefill_attention(q, kc, vc, bt, starts, ctx, d ** -0.5),
                    ops.paged_attention_decode(q[-1:], kc, vc, bt, ctx, d ** -0.5, None, 1)])
    for a, b in zip(*got):
        assert torch.equal(a, b) and a.any()
    assert not big[0][:-5].any() and not big[1][:-5].any()


def test_on_another_stream(gpu):
    """Work on a stream that is not the default one, behind work that it waits for."""
    q, kc, vc, bt, totals = _attention_case(5, 8, 2, 128, 32, torch.bfloat16, [1] * 4, [600, 31, 32, 5])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a = [t.to(gpu, non_blocking=True) for t in (q, kc, vc, bt, torch.tensor(totals, dtype=torch.int32))]
        got = ops.paged_attention_decode(*a, 128 ** -0.5, None, 4)
    side.synchronize()
    _check_attention(got.cpu(), q, kc, vc, bt, [1] * 4, totals, 128 ** -0.5)


@pytest.mark.parametrize("model", ["tiny-llama", "tiny-qwen3"])
def test_engine(gpu, model):
    """--kv-cache-dtype fp4 through the engine: as long as decode by graphs and eagerly choose the same tokens, their log
    probabilities differ by the products' rounding; first tokens are among the five likeliest of the 16-bit cache's run."""
    from kubernetes_gpu_cluster_amd.engine.llm_engine import LLM
    from kubernetes_gpu_cluster_amd.engine.sequence import SamplingParams
    prompts = [[5 + i, 6, 7, 8, 9] * 9 for i in range(3)]
    sp = SamplingParams(temperature=0, max_tokens=12, ignore_eos=True, logprobs=5)
    outs = []
    for kvd, eager in (("auto", False), ("fp4", False), ("fp4", True)):
        llm = LLM(model, device="cuda", dtype="bfloat16", random_init=True, seed=2, max_model_len=256, max_num_seqs=4,
                  max_num_batched_tokens=64, kv_cache_dtype=kvd, enforce_eager=eager)
        r = llm.engine.executor.runner
        if kvd == "fp4":
            assert r.kv.dtype == torch.uint8
        outs.append(llm.generate(prompts, sp))
        assert (r.stats["graph_steps"] > 0) == (not eager)
        llm.shutdown()
    for a, b in zip(outs[0], outs[1]):
        assert b.logprobs[0][0] in [t for t, _ in a.logprobs[0][2]]
    for a, b in zip(outs[1], outs[2]):
        for i in range(12):
            # logits below 8 in bf16, by other products on either side: two roundings of 2^-8 * 8 each
            assert abs(a.logprobs[i][2][0][1] - b.logprobs[i][2][0][1]) < 0.125
            if a.output_token_ids[i] != b.output_token_ids[i]:
                break


# ------------------------------------------------------------------ refusals
def test_refusals(gpu):
    bf, d = torch.bfloat16, 128
    kc = torch.zeros(ops.kv4_cache_shape(4, 2, 16, d), dtype=torch.uint8, device=gpu)
    q = torch.zeros(3, 4, d, dtype=bf, device=gpu)
    bt = torch.zeros(3, 2, dtype=torch.int32, device=gpu)
    n = torch.ones(3, dtype=torch.int32, device=gpu)
    table = torch.zeros(8, d, device=gpu)
    x = torch.zeros(3, 8 * d, dtype=bf, device=gpu)
    pos = torch.zeros(3, dtype=torch.int64, device=gpu)

    def no(what, f, *a, **k):
        with pytest.raises((RuntimeError, ValueError), match=what):
            f(*a, **k)
    dec, pre, wr = ops.paged_attention_decode, ops.prefill_attention, ops.rope_kv_write
    no("own scales", dec, q, kc, kc, bt, n, 1.0, k_scale=0.5)
    no("own scales", pre, q, kc, kc, bt[:1], n[:2], n[:1], 1.0, v_scale=2.0)
    no("own scales", wr, x, pos, table, kc, kc, pos, 4, 2, d, k_scale=0.5)
    no("dtype mismatch", dec, q, kc, kc.view(torch.int8), bt, n, 1.0)
    no("contiguous", dec, q, kc[:, :, :, :60], kc[:, :, :, :60], bt, n, 1.0)
    no("contiguous", dec, q, kc.transpose(0, 1), kc.transpose(0, 1), bt, n, 1.0)
    no("4-bit cache", dec, q[:, :, :64].contiguous(), kc, kc, bt, n, 1.0)
    no("bf16/f16", dec, q.float(), kc, kc, bt, n, 1.0)
    no("block_size", dec, q, kc[:, :, :8].contiguous(), kc[:, :, :8].contiguous(), bt, n, 1.0)
    odd = torch.zeros(ops.kv4_cache_shape(4, 2, 24, d), dtype=torch.uint8, device=gpu)
    no("power of two", dec, q, odd, odd, bt, n, 1.0)
    no("GQA", dec, torch.zeros(3, 34, d, dtype=bf, device=gpu), kc, kc, bt, n, 1.0)
    no("GQA", dec, torch.zeros(3, 3, d, dtype=bf, device=gpu), kc, kc, bt, n, 1.0)
    no("block_tables", dec, q, kc, kc, bt.long(), n, 1.0)
    no("block_tables", dec, q, kc, kc, bt[:2], n, 1.0)
    no("ctx_lens", dec, q, kc, kc, bt, n[:2], 1.0)
    no("different device", dec, q, kc, kc, bt.cpu(), n, 1.0)
    no("different device", dec, q, kc, kc.cpu(), bt, n, 1.0)
    no("no pages", dec, q, kc[:0], kc[:0], bt, n, 1.0)
    no("query_start_loc", pre, q, kc, kc, bt[:1], n, n[:1], 1.0, n, n)
    no("seq_lens", pre, q, kc, kc, bt[:2], n, n[:1], 1.0, n, n)
    no("work list", pre, q, kc, kc, bt[:2], n, n[:2], 1.0, n, n[:2])
    no("slices", torch.ops.kgc.prefill_attention, q, q, kc, kc, bt[:1], n[:2], n[:1], n[:1], n[:1], 1.0, 1.0, 1.0, 0,
       torch.zeros(12 * 129, device=gpu))
    wide = (torch.zeros(4, 2, 16, d, dtype=bf, device=gpu), torch.zeros(4, 2, 2, d, 8, dtype=bf, device=gpu))
    no("4-bit", torch.ops.kgc.prefill_attention, q, q, *wide, bt[:1], n[:2], n[:1], n[:1], n[:1], 1.0, 1.0, 1.0, 0,
       torch.zeros(12 * 130, device=gpu))
    no("head_dim", wr, x, pos, torch.zeros(8, 96, device=gpu), kc, kc, pos, 4, 2, 96)
    no("positions", wr, x, pos[:2], table, kc, kc, pos, 4, 2, d)
    no("slot_mapping", wr, x, pos, table, kc, kc, pos[:2], 4, 2, d)
    no("16-byte", wr, torch.zeros(3 * 8 * d + 4, dtype=bf, device=gpu)[4:].view(3, -1), pos, table, kc, kc, pos, 4, 2, d)
    p2 = pos.expand(2, 3).contiguous()
    no("sections of", wr, x, p2, table, kc, kc, pos, 4, 2, d, sections=(30, 30))
    no("1 to 4", wr, x, pos.expand(5, 3), table, kc, kc, pos, 4, 2, d, sections=(30, 30, 1, 1, 2))
    no("0 to d / 2", wr, x, p2, table, kc, kc, pos, 4, 2, d, sections=(-1, 65))
    no(r"\[sections, T\]", wr, x, pos, table, kc, kc, pos, 4, 2, d, sections=(32, 32))
    no("rotated head", wr, x, p2, table, kc, kc, pos, 4, 2, d, sections=(32, 32), use_rope=False)
    no("empty cos_sin", wr, x, p2, table[:0], kc, kc, pos, 4, 2, d, sections=(32, 32))
    no("write q too", ops.kv_write_rope, x, pos, table, kc, kc, pos, 4, 2, d)
    no("4-D / v_cache 5-D", ops.prefill_attention_rope, x, table, kc, kc, bt[:1], n[:2], n[:1], 1.0, 4, d, n[:1], n[:1])
    no("slots int64", ops.kv4_read, kc, pos.int(), bf)
    no("bf16 / fp16", ops.kv4_read, kc, pos, torch.float32)
    no("4-bit cache", ops.kv4_read, kc[..., :60].contiguous(), pos, bf)


def test_a_cache_without_heads_is_refused(gpu):
    d = 128
    kc = torch.zeros(ops.kv4_cache_shape(4, 1, 16, d), dtype=torch.uint8, device=gpu)[:, :0].contiguous()
    pos = torch.zeros(3, dtype=torch.int64, device=gpu)
    with pytest.raises(RuntimeError, match="no heads"):
        ops.kv4_read(kc, pos, torch.bfloat16)
    with pytest.raises(RuntimeError, match="no heads"):
        ops.rope_kv_write(torch.zeros(3, 4 * d, dtype=torch.bfloat16, device=gpu), pos, torch.zeros(8, d, device=gpu),
                          kc, kc.clone(), pos, 4, 0, d)


@pytest.mark.parametrize("nq,nkv", [(0, 2), (4, 0), (0, 0)])
def test_queries_without_heads_are_refused(gpu, nq, nkv):
    d = 128
    kc = torch.zeros(ops.kv4_cache_shape(4, max(nkv, 1), 16, d), dtype=torch.uint8, device=gpu)[:, :nkv].contiguous()
    q = torch.zeros(3, nq, d, dtype=torch.bfloat16, device=gpu)
    bt = torch.zeros(3, 64, dtype=torch.int32, device=gpu)
    n = torch.ones(3, dtype=torch.int32, device=gpu)
    for z in (1, 2):
        with pytest.raises(RuntimeError, match="GQA group|4-bit cache"):
            ops.paged_attention_decode(q, kc, kc, bt, n, 1.0, None, z)
    with pytest.raises(RuntimeError, match="GQA group|4-bit cache"):
        ops.prefill_attention(q, kc, kc, bt, torch.arange(4, dtype=torch.int32, device=gpu), n, 1.0)


@pytest.mark.parametrize("z", [1, 4])
def test_numbers_that_would_wrap(gpu, z):
    """Work items, row ranges and lengths whose products or differences leave 32 bits are left out like others that
    are none: 2^24 blocks of 128 rows are -2^31, 2^25 are 0."""
    if ops.DEBUG:
        pytest.skip("the bounds-checking build reports them")
    low = -2 ** 31
    new, old = [20, 40], [100, 300]
    q, kc, vc, bt, totals = _attention_case(9, 4, 2, 64, 32, torch.bfloat16, new, old)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)   # noqa: E731
    qg, a = q.to(gpu), [t.to(gpu) for t in (kc, vc, bt)]
    parts = torch.empty(z * q.numel() // 64 * 66, device=gpu)

    def run(starts, n, ws, wm):
        out = torch.full_like(qg, 7)
        torch.ops.kgc.prefill_attention(out, qg, *a, starts, n, ws, wm, 0.125, 1.0, 1.0, 0, parts)
        return out
    # (the second sequence's only true item comes first; items of block 0, again, would write the same rows)
    out = run(_starts(new).to(gpu), i32(*totals), i32(1, 0, 0, 0, 0), i32(0, 1 << 24, 1 << 25, 2 ** 31 - 1, (1 << 24) + 1))
    assert (out[:20] == 7).all()
    _check_attention(out[20:].cpu(), q[20:], kc, vc, bt[1:], new[1:], totals[1:], 0.125)
    for starts, n in ((i32(low, low + 20, 60), i32(*totals)), (i32(5, low, low + 3), i32(*totals)), (i32(0, 2 ** 31 - 1, 60), i32(*totals)),
                      (_starts(new).to(gpu), i32(low, low + 7))):
        assert (run(starts, n, i32(0, 1), i32(0, 0)) == 7).all()
    dec = ops.paged_attention_decode(torch.stack([q[0], q[59]]).to(gpu), *a, i32(low, totals[1]), 0.125, None, z)
    assert not dec[0].any()
    _check_attention(dec[1:].cpu(), q[59:], kc, vc, bt[1:], [1], totals[1:], 0.125)


def test_launches_up_to_their_limit(gpu):
    """2^24 workgroups of 256 prompt threads are more than a launch takes: refused; the longest list below them runs."""
    new, old, nq = [20], [100], 16
    q, kc, vc, bt, totals = _attention_case(9, nq, 1, 64, 32, torch.bfloat16, new, old)
    a = [t.to(gpu) for t in (q, kc, vc, bt, _starts(new), torch.tensor(totals, dtype=torch.int32))]
    items = (1 << 24) // nq
    ws, wm = torch.full((items,), -1, dtype=torch.int32, device=gpu), torch.zeros(items, dtype=torch.int32, device=gpu)
    with pytest.raises(RuntimeError, match="too many work items"):
        ops.prefill_attention(*a, 0.125, ws, wm)
    ws[-2] = 0
    out = torch.full_like(a[0], 7)
    ops.prefill_attention(*a, 0.125, ws[:-1], wm[:-1], out=out)
    _check_attention(out.cpu(), q, kc, vc, bt, new, totals, 0.125)
    wide = torch.zeros(1, (1 << 25) + 1, dtype=torch.int32, device=gpu)
    with pytest.raises(RuntimeError, match="2\\^30"):
        ops.paged_attention_decode(a[0][:1], *a[1:3], wide, a[5], 0.125)


@pytest.mark.parametrize("scale", [0.0, -0.125, float("nan"), float("inf"), 1e-60, 1e60])
def test_scales_of_prompts(gpu, scale):
    """The prompt kernel scales behind the mask and the maximum: a scale that is not above zero, in 32 bits, is refused.
    Decode scales first and takes those that are numbers."""
    new, old = [40, 1], [30, 70]
    q, kc, vc, bt, totals = _attention_case(3, 4, 2, 64, 32, torch.bfloat16, new, old)
    a = [t.to(gpu) for t in (q, kc, vc, bt, _starts(new), torch.tensor(totals, dtype=torch.int32))]
    with pytest.raises(RuntimeError, match="above zero"):
        ops.prefill_attention(*a, scale)
    with pytest.raises(RuntimeError, match="above zero"):
        ops.prefill_attention(*a, scale, out=torch.empty_like(a[0]))
    if abs(scale) < 1:
        last = q[[39, 40]]
        got = ops.paged_attention_decode(last.to(gpu), *a[1:4], a[5], scale)
        _check_attention(got.cpu(), last, kc, vc, bt, [1, 1], totals, scale)


@pytest.mark.parametrize("cache", ["auto", "fp8", "fp4"])
def test_axes_refuse_strides_and_norms_of_other_kinds(gpu, cache):
    """Slots are read one after the other, norm weights as numbers of q's type on its device, whatever the pages hold."""
    d, T, bf = 64, 8, torch.bfloat16
    if cache == "fp4":
        kc, vc = (torch.zeros(ops.kv4_cache_shape(2, 1, 16, d), dtype=torch.uint8, device=gpu) for _ in range(2))
    else:
        t = torch.float8_e4m3fn if cache == "fp8" else bf
        kc, vc = torch.zeros(2, 1, 16, d, device=gpu).to(t), torch.zeros(2, 1, 2, d, 8, device=gpu).to(t)
    x = torch.randn(T, 4 * d, device=gpu).to(bf)
    table = ref.rope_cos_sin_cache(d, 20, 10000.0).to(gpu)
    slots = torch.arange(2 * T, device=gpu)
    pos, w = torch.zeros(2, T, dtype=torch.int64, device=gpu), torch.ones(d, dtype=bf, device=gpu)

    def write(slots, *norms, pos=pos, sections=(16, 16)):
        return ops.rope_kv_write(x, pos, table, kc, vc, slots, 2, 1, d, *norms, sections=sections)
    for bad in ((slots[::2],), (slots[:T], w.cpu(), w), (slots[:T], w, w.float()), (slots[:T], w, w[:8]), (slots[:T], w, None),
                (slots[:T], torch.ones(2 * d, dtype=bf, device=gpu)[::2], w)):
        with pytest.raises(RuntimeError, match="contiguous|norm weights"):
            write(*bad)
    with pytest.raises(RuntimeError, match="contiguous"):
        write(slots[:T], pos=slots[::2], sections=None)
    with pytest.raises(RuntimeError, match="contiguous"):
        write(slots[::2], pos=slots[:T], sections=None)
    assert not kc.float().any() and not vc.float().any()
    write(slots[:T], w, w)
    assert kc.float().any() and vc.float().any()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("T", [4, 40])
def test_keys_beside_borders(gpu, dt, T):
    """Keys whose rotation is nearer to a border of two codes than 64 bits hold have the code of the exact sum."""
    x, table, want, e = oracle.keys_beside_borders()
    i = torch.arange(T) % len(x)
    qkv = torch.zeros(T, 3, 64)
    qkv[:, 1] = x[i]
    kc, vc = (torch.zeros(ops.kv4_cache_shape(2, 1, 32, 64), dtype=torch.uint8, device=gpu) for _ in range(2))
    slots = torch.arange(T, device=gpu)
    ops.rope_kv_write(qkv.to(dt).view(T, -1).to(gpu), slots * 0, table.to(gpu), kc, vc, slots, 1, 1, 64)
    assert torch.equal(ops.kv4_read(kc, slots, dt)[:, 0].double().cpu(), want[i])
    scales = ref.kv4_parts(kc.cpu())[1].transpose(1, 2).flatten(0, 1)[:T, 0]
    assert torch.equal(scales.double() - 127, e[i])


@pytest.mark.parametrize("dt", DT)
def test_rotated_infinities_and_nan(gpu, dt):
    """Sums beyond 32 bits, of infinities and of NaN are stored as the CPU stores them."""
    T, d, big = 6, 64, torch.finfo(dt).max
    x = torch.randn(T, 3, d, generator=_gen(8))
    x[0, 1, 3], x[1, 1, 35], x[2, 1, 3], x[3, 1, 3], x[3, 1, 35] = float("inf"), -float("inf"), float("nan"), big, big
    x[4, 1, 3], x[4, 1, 35] = float("inf"), float("inf")
    x = x.to(dt).view(T, -1)
    table = torch.cat([torch.full((32,), 2.0 ** 125), torch.full((32,), -2.0 ** 126)])[None]
    table[0, 8:16], table[0, 40:48] = 2.0 ** -140, 2.0 ** -149           # below 32 bits
    got = []
    for dev in (torch.device("cpu"), gpu):
        kc, vc = (torch.zeros(ops.kv4_cache_shape(1, 1, 16, d), dtype=torch.uint8, device=dev) for _ in range(2))
        slots = torch.arange(T, device=dev)
        ops.rope_kv_write(x.to(dev), slots * 0, table.to(dev), kc, vc, slots, 1, 1, d)
        got.append(ops.kv4_read(kc, slots, dt).cpu())
    assert torch.equal(*got) and got[0].isfinite().all()


def _launched(f):
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        f()
        torch.cuda.synchronize()
    return [e.key for e in prof.key_averages() if e.device_type == torch.autograd.DeviceType.CUDA]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("S,norms", [(0, False), (3, False), (8, True), (0, True)])
def test_decode_step_with_row_scales(gpu, dt, S, norms):
    """A decode step's projection times a number per row before its rounding, in the launch that rotates: as the same step
    over the rows that fp32 sums, the product and one rounding give, and in two launches."""
    g, B, nq, nkv, d, bs = _gen(S + 17), 9, 8, 2, 128, 32
    x = torch.randn(max(S, 1), B, (nq + 2 * nkv) * d, generator=g)
    x = x if S else x[0].to(dt)
    r = torch.rand(B, generator=g) + 0.5
    rows = x.float() if not S else x[0]
    for z in range(1, S):
        rows = rows + x[z]
    rows = (rows * r[:, None]).to(dt)
    ctx = [1 + 29 * i for i in range(B)]
    bt, nb = oracle.tables(g, ctx, bs)
    kc, vc = (oracle.random_cache(g, nb, nkv, bs, d, dt) for _ in range(2))
    slots = torch.tensor([int(bt[i, (n - 1) // bs]) * bs + (n - 1) % bs for i, n in enumerate(ctx)])
    w = [torch.rand(d, generator=g).add(0.5).to(dt).to(gpu) for _ in range(2)] if norms else [None, None]
    pos, table = torch.tensor(ctx, device=gpu) - 1, ref.rope_cos_sin_cache(d, 300, 10000.0).to(gpu)

    def step(qkv, caches, **k):
        return ops.paged_attention_decode_rope(qkv, pos, table, *caches, slots.to(gpu), nq, nkv, d, bt.to(gpu),
                                               (pos + 1).int(), d ** -0.5, *w, dtype=dt, **k)
    got, want = ([c.to(gpu) for c in (kc, vc)] for _ in range(2))
    a, b = step(x.to(gpu), got, row_scale=r.to(gpu)), step(rows.to(gpu), want)
    assert torch.equal(a, b) and all(torch.equal(p, q) for p, q in zip(got, want))
    xg, rg = x.to(gpu), r.to(gpu)
    names = _launched(lambda: step(xg, got, row_scale=rg))
    assert sum("kv4_" in n for n in names) == 2 and not any("reduce" in n for n in names), names


def test_row_scales_refused(gpu):
    d, T, bf = 128, 3, torch.bfloat16
    kc, vc = (torch.zeros(ops.kv4_cache_shape(2, 1, 16, d), dtype=torch.uint8, device=gpu) for _ in range(2))
    x, table = torch.zeros(T, 4 * d, dtype=bf, device=gpu), torch.zeros(8, d, device=gpu)
    pos, n = torch.arange(T, device=gpu), torch.ones(T, dtype=torch.int32, device=gpu)
    bt, r = torch.zeros(T, 1, dtype=torch.int32, device=gpu), torch.ones(2 * T, device=gpu)
    for bad in (r, r[::2], r[:T].double(), r[:T].cpu()):
        with pytest.raises(RuntimeError, match="row_scale"):
            ops.paged_attention_decode_rope(x, pos, table, kc, vc, pos, 2, 1, d, bt, n, 1.0, row_scale=bad)
    wide = torch.zeros(2, 1, 16, d, dtype=bf, device=gpu), torch.zeros(2, 1, 2, d, 8, dtype=bf, device=gpu)
    with pytest.raises(RuntimeError, match="4-bit caches"):
        torch.ops.kgc.rope_kv_write(x, pos, table, torch.empty(T, 2, d, dtype=bf, device=gpu), *wide, pos, None, None, 2, 1, d,
                                    1e-6, True, 1.0, 1.0, None, r[:T])
    with pytest.raises(RuntimeError, match="without sections"):
        torch.ops.kgc.rope_kv_write(x, pos[None], table, torch.empty(T, 2, d, dtype=bf, device=gpu), kc, vc, pos, None, None, 2, 1,
                                    d, 1e-6, True, 1.0, 1.0, [64], r[:T])


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("B,z", [(3, 1), (3, 3), (70, 1)])
def test_values_that_are_alike_come_back(gpu, dt, B, z):
    """Weights add up to one as they are rounded: with values that are all 1 the result is 1, whatever the weights' rounding.
    Of every 32 keys 31 have a weight just below the middle between a half and the type's next number.  (Numerator and
    denominator are sums of the same 400 or fewer numbers: 2^-15 apart at most, an eighth of half of fp16's step.)"""
    n, d, u = 400, 64, torch.finfo(dt).eps / 2
    kc, vc = (torch.zeros(ops.kv4_cache_shape(14, 1, 32, d), dtype=torch.uint8, device=gpu) for _ in range(2))
    for c in (kc, vc):
        ref.kv4_parts(c)[1].fill_(127)
    ref.kv4_parts(vc)[0].fill_(0x22)
    ref.kv4_parts(kc)[0][:, :, 1:, 0] = 0xA                   # -1 in the first element
    q = torch.zeros(B, 2, d, dtype=dt, device=gpu)
    q[..., 0] = 1
    scale = math.log(2) - math.log1p(0.98 * u)
    bt = torch.arange(14, dtype=torch.int32, device=gpu).expand(B, 14).contiguous()
    ctx = torch.tensor([n, 200, 333] + [n - i for i in range(B - 3)], dtype=torch.int32, device=gpu)
    assert (ops.paged_attention_decode(q, kc, vc, bt, ctx, scale, None, z) == 1).all()
    starts = torch.arange(B + 1, dtype=torch.int32, device=gpu)
    assert (ops.prefill_attention(q, kc, vc, bt, starts, ctx, scale) == 1).all()


@pytest.mark.parametrize("z", [1024, 1025, 5000])
def test_decode_of_more_slices_than_a_merge_takes(gpu, z):
    """Slices beyond the merge's 1024 are 1024, as over the wider caches; 0 are refused."""
    ctx = [700, 1, 300]
    q, kc, vc, bt, _ = _attention_case(4, 4, 2, 64, 32, torch.bfloat16, [1] * 3, [c - 1 for c in ctx])
    a = [t.to(gpu) for t in (q, kc, vc, bt, torch.tensor(ctx, dtype=torch.int32))]
    got = ops.paged_attention_decode(*a, 0.125, None, z)
    _check_attention(got.cpu(), q, kc, vc, bt, [1] * 3, ctx, 0.125)
    with pytest.raises(RuntimeError, match="Z"):
        ops.paged_attention_decode(*a, 0.125, None, 0)


# ------------------------------------------------------------------ the forms that large steps take
def _ran(names, kernel, *args):
    """Whether a kernel's form with these last template arguments is among the launched ones; the profiler has names mangled or
    plain (the 16-bit types are beyond some demanglers)."""
    raw = "".join(f"Lb{int(a)}E" if isinstance(a, bool) else f"Li{a}E" for a in args) + "EEv"
    plain = ", ".join(str(a).lower() for a in args) + ">"
    return any(kernel in n and (raw in n or plain in n) for n in names)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("nq,nkv,d,bs,T,sections", [
    (32, 8, 128, 32, 2800, None),
    (32, 8, 128, 32, 2733, (10, 9, -1)),
    (15, 5, 128, 16, 5300, None),                              # 25 heads: the last four are one
    (15, 5, 128, 64, 5250, (5, -1)),
    (12, 12, 64, 32, 7300, None),
    (13, 5, 64, 32, 11500, (-1,)),                             # 23 heads: the last four are three
])
def test_write_of_many_rows(gpu, dt, nq, nkv, d, bs, T, sections):
    """More than 4096 workgroups of a head per thread: four heads per thread (kv4_cache.hip kv4_write_dispatch)."""
    names = _launched(lambda: test_write(gpu, dt, nq, nkv, d, bs, T, sections, 0))
    assert _ran(names, "kv4_write_kernel", True, False, sections is not None, 4, False), names


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rope,norms", [(True, True), (False, True), (False, False)])
def test_write_of_many_rows_normed_and_unrotated(gpu, dt, rope, norms):
    """Four heads per thread write what a head per thread writes: the same rows in one call and in calls of 500."""
    g, nq, nkv, d, bs, T = _gen(3), 30, 7, 128, 32, 3500
    x = torch.randn(T, (nq + 2 * nkv) * d, generator=g).to(dt).to(gpu)
    w = [torch.rand(d, generator=g).add(0.5).to(dt).to(gpu) for _ in range(2)] if norms else [None, None]
    pos, table = torch.randint(0, 300, (T,), generator=g).to(gpu), ref.rope_cos_sin_cache(d, 300, 10000.0).to(gpu)
    slots = torch.randperm(T + 60, generator=g)[:T].to(gpu)
    slots[5] = -1
    got = []

    def write(step):
        caches = [torch.zeros(ops.kv4_cache_shape(-(-(T + 60) // bs), nkv, bs, d), dtype=torch.uint8, device=gpu) for _ in range(2)]
        q = [ops.rope_kv_write(x[a:a + step], pos[a:a + step], table, *caches, slots[a:a + step], nq, nkv, d, *w, use_rope=rope)
             for a in range(0, T, step)]
        got.append([torch.cat(q), *caches])
    for step, heads in ((T, 4), (500, 1)):
        names = _launched(lambda: write(step))
        assert _ran(names, "kv4_write_kernel", rope, False, False, heads, False), names
    assert all(torch.equal(a, b) for a, b in zip(*got)) and got[0][1].any()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("nkv,d,n", [(8, 128, 8200), (12, 64, 10950), (1, 128, 65601), (8, 128, 8190)])
def test_read_of_many_rows(gpu, dt, nkv, d, n):
    """2^20 pieces of 8 elements and more are read four per thread (the last case: just fewer)."""
    g = _gen(n)
    c = oracle.random_cache(g, 70, nkv, 16, d, dt)
    slots = torch.randint(0, 70 * 16, (n,), generator=g)
    slots[3], slots[n // 2], slots[n - 1] = -1, 70 * 16, 1 << 40
    assert (n * nkv * (d // 8) >= 1 << 20) == (n != 8190)
    got = ops.kv4_read(c.to(gpu), slots.to(gpu), dt).cpu()
    assert torch.equal(got, ref.kv4_read(c, slots, dt))


def _attention_wanted(q, kc, vc, bt, new, totals, scale):
    """What _check_attention compares with, once for several calls: results and how far off, [rows, heads, d]."""
    nq, nkv = q.shape[1], kc.shape[1]
    want, tol, at = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64), 0
    for i, (m, n) in enumerate(zip(new, totals)):
        seen = torch.arange(n)[None] <= torch.arange(n - m, n)[:, None]
        for h in range(nkv if n else 0):
            k, v = (oracle.rows(c, bt[i], n, h, q.shape[2]) for c in (kc, vc))
            g = nq // nkv                                     # a group's rows at once
            rows = q[at:at + m, h * g:(h + 1) * g].transpose(0, 1).flatten(0, 1)
            o, t = oracle.attend(rows, k, v, scale, seen.repeat(g, 1), q.dtype)
            for to, x in ((want, o), (tol, t)):
                to[at:at + m, h * g:(h + 1) * g] = x.view(g, m, -1).transpose(0, 1)
        at += m
    return want, tol


# The waves of a workgroup go by the (sequence, kv head) pairs: fewer than 64 four, to 511 eight, to 1023 four, to 1535 two, then one
DECODE_FORMS = [
    # waves, q heads, kv heads, head, page, contexts
    (8, 32, 8, 128, 32, [700, 1, 0, 33, 320, 64, 511, 2300, 90]),
    (8, 16, 1, 128, 16, [1 + 37 * i % 500 for i in range(66)]),
    (8, 6, 2, 128, 64, [700 - 19 * i for i in range(36)]),
    (8, 10, 2, 64, 32, [2 + 41 * i % 800 for i in range(40)] + [2500]),
    (4, 32, 8, 128, 32, [1 + 53 * i % 900 for i in range(70)] + [2100]),
    (4, 15, 5, 64, 16, [600 - 5 * i for i in range(105)]),
    (2, 32, 8, 128, 32, [61 * i % 700 for i in range(129)] + [2300]),
    (2, 12, 4, 64, 32, [1 + 43 * i % 500 for i in range(260)]),
    (1, 32, 8, 128, 32, [59 * i % 650 for i in range(199)] + [2200]),
    (1, 12, 2, 128, 16, [1 + 31 * i % 300 for i in range(770)]),
    (1, 8, 4, 64, 64, [47 * i % 400 for i in range(399)] + [2400]),
]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("waves,nq,nkv,d,bs,ctx", DECODE_FORMS)
def test_decode_by_waves(gpu, dt, waves, nq, nkv, d, bs, ctx):
    """Every number of waves, over contexts that take several turns of their loops, with heads that share a kv head, whole and
    in slices."""
    B = len(ctx)
    q, kc, vc, bt, _ = _attention_case(B + d, nq, nkv, d, bs, dt, [1] * B, [c - 1 for c in ctx])
    want, tol = _attention_wanted(q, kc, vc, bt, [1] * B, ctx, d ** -0.5)
    a = [t.to(gpu) for t in (q, kc, vc, bt, torch.tensor(ctx, dtype=torch.int32))]
    rule = ops.decode_grid_z(B, nkv, max(ctx), cache_dtype=torch.uint8)
    assert ops.kv4_decode_waves(B * nkv) == waves
    for z in sorted({1, 2, 5, rule}):
        got = []
        names = _launched(lambda: got.append(ops.paged_attention_decode(*a, d ** -0.5, None, z)))
        assert _ran(names, "kv4_decode_kernel", d, waves) and any("paged_decode_reduce" in n for n in names) == (z > 1), names
        assert ((got[0].cpu().double() - want).abs() <= tol).all(), z


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("nq,nkv,d,bs,new,old,heads", [
    (32, 8, 128, 32, [300, 33, 1], [2000, 700, 0], 4),
    (12, 12, 64, 16, [301, 280, 226], [1500, 1400, 20], 1),
    (12, 6, 128, 64, [290, 129, 140], [0, 1900, 450], 2),
    (24, 2, 64, 32, [200, 127, 1, 260], [1100, 90, 800, 0], 4),
])
@pytest.mark.parametrize("z", [8, 13, 32])
def test_prompts_in_slices_by_many_workgroups(gpu, dt, nq, nkv, d, bs, new, old, heads, z):
    """Slices that come to more than two workgroups per CU (512 here): one LDS buffer per tile."""
    if torch.cuda.get_device_properties(gpu).multi_processor_count != 256:
        pytest.skip("lines for 256 CUs")
    assert sum(-(-n // 128) for n in new) * nq * z > 512
    names = _launched(lambda: test_prompts_in_slices(gpu, dt, nq, nkv, d, bs, new, old, z))
    assert _ran(names, "kv4_prefill_kernel", heads, 1) and any("kv4_prefill_merge" in n for n in names), names


def test_slices_that_the_rule_gives(gpu):
    """The public call's own slices where they come to many workgroups, with a result of its own and one of the caller's."""
    new, old, nq, nkv, d = [301, 264, 227], [7000, 6500, 3000], 12, 12, 64
    q, kc, vc, bt, totals = _attention_case(5, nq, nkv, d, 32, torch.float16, new, old)
    assert ops.kv4_prefill_slices(sum(new), 3, nq, nkv, d, max(totals)) > 1
    want, tol = _attention_wanted(q, kc, vc, bt, new, totals, d ** -0.5)
    a = [t.to(gpu) for t in (q, kc, vc, bt, _starts(new), torch.tensor(totals, dtype=torch.int32))]
    for out in (None, torch.full_like(a[0], 7)):
        got = []
        names = _launched(lambda: got.append(ops.prefill_attention(*a, d ** -0.5, out=out)))
        assert any("kv4_prefill_merge" in n for n in names) and (out is None or got[0] is out)
        assert ((got[0].cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("cache", ["auto", "fp8"])
@pytest.mark.parametrize("nq,nkv,d,bs,T,sections,by_rows", [
    (12, 12, 64, 32, 1400, (8, 12, 12), True),
    (12, 12, 64, 32, 1300, (8, 12, 12), False),               # fewer than 3M elements: a launch
    (25, 5, 64, 16, 2001, (3, 0, 20, 9), True),               # 30 heads of q and k: the last four are two
    (5, 1, 64, 24, 7100, (32,), True),
    (33, 3, 128, 16, 700, (50, 14), True),
])
def test_axes_of_many_rows(gpu, dt, cache, nq, nkv, d, bs, T, sections, by_rows):
    """q and k by rows and v by 8-row groups, from 3 * 2^20 elements on, as the one-position kernel turns each axis's pairs."""
    g, t = _gen(T), torch.float8_e4m3fn if cache == "fp8" else dt
    nb = T // bs + 3
    mk = lambda: (torch.zeros(nb, nkv, bs, d).to(t).to(gpu), torch.zeros(nb, nkv, bs // 8, d, 8).to(t).to(gpu))   # noqa: E731
    x = torch.randn(T, (nq + 2 * nkv) * d, generator=g).to(dt).to(gpu)
    table = ref.rope_cos_sin_cache(d, 90, 10000.0)
    pos = torch.randint(-5, 99, (len(sections), T), generator=g)
    slots = torch.arange(T) + 5                               # runs that start in an 8-key group, one that ends in one, and padding
    slots[100:] += 3
    slots[-3:] = -1
    slots = slots.to(gpu)
    kc, vc = mk()
    q = []
    names = _launched(lambda: q.append(ops.rope_kv_write(x, pos.to(gpu), table.to(gpu), kc, vc, slots, nq, nkv, d,
                                                         sections=sections)))
    assert any("rope_rows_kernel" in n for n in names) == any("kv_group_kernel" in n for n in names) == by_rows, names
    for a, n in enumerate(sections):
        rows = table[pos[a].clamp(0, 89)].contiguous().to(gpu)
        k2, v2 = mk()
        q2 = ops.rope_kv_write(x, torch.arange(T, device=gpu), rows, k2, v2, slots, nq, nkv, d)
        i = torch.arange(sum(sections[:a]), sum(sections[:a + 1]), device=gpu)
        i = torch.cat([i, i + d // 2])
        assert torch.equal(q[0][..., i], q2[..., i])
        assert torch.equal(kc.float()[..., i], k2.float()[..., i]) and torch.equal(vc.float(), v2.float())
    assert vc.float().any() and kc.float().any()


@pytest.mark.parametrize("eager", [False, True])
def test_engine_of_learned_positions(gpu, eager):
    """OPT over a 4-bit cache: heads of 64, one q head per kv head, nothing rotated.  Prompts in chunks and decode steps run, and
    every layer's pages hold what was written."""
    from kubernetes_gpu_cluster_amd.engine.llm_engine import LLM
    from kubernetes_gpu_cluster_amd.engine.sequence import SamplingParams
    from kubernetes_gpu_cluster_amd.models import configs
    configs.PRESETS["opt-125m-two"] = configs.PRESETS["opt-125m"].shrink(name="opt-125m-two", num_layers=2)
    try:
        llm = LLM("opt-125m-two", device="cuda", dtype="float16", random_init=True, seed=2, max_model_len=256, max_num_seqs=4,
                  max_num_batched_tokens=64, num_gpu_blocks_override=64, kv_cache_dtype="fp4", enforce_eager=eager)
    finally:
        del configs.PRESETS["opt-125m-two"]
    r = llm.engine.executor.runner
    assert r.kv.dtype == torch.uint8 and r.kv.shape[:2] == (2, 2)
    outs = llm.generate([[5 + i, 6, 7, 8, 9] * 9 for i in range(3)],
                        SamplingParams(temperature=0, max_tokens=6, ignore_eos=True, logprobs=5))
    assert (r.stats["graph_steps"] > 0) == (not eager)
    for o in outs:
        assert len(o.output_token_ids) == 6 and all(math.isfinite(p) for step in o.logprobs for _, p in step[2])
    # 3 prompts of 45 tokens and five of their answers' six: rows with a scale of their own
    for layer in r.kv:
        for c in layer:
            assert int((ref.kv4_parts(c)[1] != 0).all(-1).all(1).sum()) == 3 * 50
    llm.shutdown()


@pytest.mark.parametrize("cache", ["auto", "fp8"])
@pytest.mark.parametrize("T,slices", [(40, 0), (40, 2), (1400, 0)])
def test_axes_leave_out_slots_beyond_the_pool(gpu, cache, T, slices):
    """As the 4-bit write does, in one launch and by rows and 8-row groups; pages behind the pool in the same allocation stay."""
    if ops.DEBUG:
        pytest.skip("the bounds-checking build reports them")
    g, dt, nq, nkv, d, bs = _gen(6), torch.bfloat16, 12, 12, 64, 32
    t, nb = torch.float8_e4m3fn if cache == "fp8" else dt, T // bs + 2
    x = torch.randn(max(slices, 1), T, (nq + 2 * nkv) * d, generator=g)
    x = x.to(gpu) if slices else x[0].to(dt).to(gpu)
    table = ref.rope_cos_sin_cache(d, 90, 10000.0).to(gpu)
    pos = torch.randint(0, 90, (2, T), generator=g).to(gpu)
    good = torch.arange(T) + 3
    bad = good.clone()
    for i, s in ((5, nb * bs), (9, nb * bs + 17), (17, 1 << 40), (T - 1, -7), (T - 2, 2 ** 31 + 5)):
        bad[i], good[i] = s, -1
    got = []
    for slots in (good, bad):
        k_all, v_all = torch.zeros(nb + 3, nkv, bs, d, device=gpu).to(t), torch.zeros(nb + 3, nkv, bs // 8, d, 8, device=gpu).to(t)
        q = ops.rope_kv_write(x, pos, table, k_all[:nb], v_all[:nb], slots.to(gpu), nq, nkv, d, dtype=dt, sections=(12, 20))
        got.append([q, k_all.float(), v_all.float()])
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert got[0][1].any() and not got[1][1][nb:].any() and not got[1][2][nb:].any()


@pytest.mark.parametrize("cache", ["auto", "fp4"])
def test_strided_positions_that_nothing_reads(gpu, cache):
    """Without rotation positions may lie anywhere: the call writes what it writes with dense ones."""
    d, T, bf = 64, 8, torch.bfloat16
    x = torch.randn(T, 4 * d, device=gpu).to(bf)
    table, pos, slots = ref.rope_cos_sin_cache(d, 20, 10000.0).to(gpu), torch.arange(2 * T, device=gpu), torch.arange(T, device=gpu)
    got = []
    for p in (pos[::2], pos[:T]):
        if cache == "fp4":
            kc, vc = (torch.zeros(ops.kv4_cache_shape(2, 1, 16, d), dtype=torch.uint8, device=gpu) for _ in range(2))
        else:
            kc, vc = torch.zeros(2, 1, 16, d, device=gpu).to(bf), torch.zeros(2, 1, 2, d, 8, device=gpu).to(bf)
        got.append([ops.rope_kv_write(x, p, table, kc, vc, slots, 2, 1, d, use_rope=False), kc, vc])
    assert all(torch.equal(a, b) for a, b in zip(*got)) and got[0][1].any()
