"""The 4-bit key / value cache and rotary positions on several axes, on the CPU: the reference ops against
64 bits, and the engine with such a cache."""
import pytest
import torch

import kv4_oracle as oracle
from kubernetes_gpu_cluster_amd import ops
from kubernetes_gpu_cluster_amd.ops import reference as ref

DT = [torch.bfloat16, torch.float16]


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("dt", DT)
def test_codes_are_the_nearest(dt):
    g = _gen()
    x = torch.randn(60, 128, generator=g).double() * torch.exp(2 * torch.randn(128, generator=g)).double()
    x[0, :32] = 0
    x[1] *= 1e-40
    x[2, 5] = 60000.0
    x[3, :32] = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6] * 4)      # ties: to the even code
    x[4, :32] = -x[3, :32] * 2 ** 9
    x[5, 0], x[5, 32] = 7.0, 7.0001                                            # where the scale changes
    want, e = oracle.nearest(x, dt)
    n, s = ref.kv4_quantize(x, dt)
    assert torch.equal(ref.kv4_dequantize(n, s).double(), want) and torch.equal(s.double() - 127, e)
    assert torch.equal(want.to(dt).double(), want)                             # a number of the type
    # half a step: a twelfth of the block's scale for small ones, 1 scale up to 7 of them
    inside = x.abs() <= 7 * 2 ** e.repeat_interleave(32, -1)
    assert ((want - x).abs() <= 2 ** e.repeat_interleave(32, -1))[inside].all()


def test_codes_of_infinities_and_nan():
    x = torch.zeros(3, 64)
    x[0, 3], x[0, 40] = float("inf"), float("nan")
    x[1, 3], x[1, 4] = -float("inf"), 1.0
    for dt, top in ((torch.bfloat16, 6 * 2.0 ** 125), (torch.float16, 6 * 2.0 ** 13)):
        v = ref.kv4_dequantize(*ref.kv4_quantize(x, dt))
        assert v[0, 3] == top and v[0, 40] == 0 and v[1, 3] == -top and v[1, 4] == 0 and not v[2].any()


@pytest.mark.parametrize("d", [64, 128])
def test_write_read_and_layout(d):
    g = _gen(1)
    dt, nkv, bs, T = torch.bfloat16, 3, 16, 21
    kc = oracle.random_cache(g, 4, nkv, bs, d, dt)
    vc, old = kc.clone(), kc.clone()
    assert kc.shape == ops.kv4_cache_shape(4, nkv, bs, d)
    qkv = torch.randn(T, (4 + 2 * nkv) * d, generator=g).to(dt)
    slots = torch.randperm(4 * bs, generator=g)[:T]
    slots[5], slots[6] = -1, 4 * bs                                            # of no page
    pos = torch.randint(0, 50, (T,), generator=g)
    table = ref.rope_cos_sin_cache(d, 50, 10000.0)
    ops.rope_kv_write(qkv, pos, table, kc, vc, slots, 4, nkv, d)
    x = qkv.double().view(T, 4 + 2 * nkv, d)
    cos, sin = oracle.cos_sin_rows(table, pos)
    k, v = oracle.nearest(oracle.rotate(x[:, 4:4 + nkv], cos, sin), dt)[0], oracle.nearest(x[:, 4 + nkv:], dt)[0]
    kept = torch.ones(4, bs, dtype=torch.bool)
    for t in range(T):
        if 0 <= slots[t] < 4 * bs:
            kept[slots[t] // bs, slots[t] % bs] = False
            for h in range(nkv):
                assert torch.equal(oracle.token(kc, int(slots[t]), h, d), k[t, h])
                assert torch.equal(oracle.token(vc, int(slots[t]), h, d), v[t, h])
    for new, was in zip(ref.kv4_parts(kc) + ref.kv4_parts(vc), ref.kv4_parts(old) * 2):
        assert torch.equal(new.transpose(1, 2)[kept], was.transpose(1, 2)[kept])
    got = ops.kv4_read(kc, slots, dt)
    there = (slots >= 0) & (slots < 4 * bs)
    assert torch.equal(got[there].double(), k[there]) and not got[~there].any()


@pytest.mark.parametrize("sections", [(32,), (8, 12, 12), (0, 5, 27), (1, 2, 3, 26)])
@pytest.mark.parametrize("cache", ["fp4", "auto", "fp8"])
def test_axes(sections, cache):
    g = _gen(2)
    dt, d, T, nq, nkv, bs = torch.bfloat16, 64, 19, 4, 2, 16
    qkv = torch.randn(T, (nq + 2 * nkv) * d, generator=g).to(dt)
    pos = torch.randint(-3, 70, (len(sections), T), generator=g)               # outside the table: its ends
    table = ref.rope_cos_sin_cache(d, 60, 10000.0)
    kc, vc = _caches(cache, 3, nkv, bs, d, dt)
    slots = torch.arange(T) + 3
    q = ops.rope_kv_write(qkv, pos, table, kc, vc, slots, nq, nkv, d, sections=sections)
    cos, sin = oracle.cos_sin_rows(table, pos, sections)
    x = qkv.double().view(T, nq + 2 * nkv, d)
    want = oracle.rotate(x[:, :nq], cos, sin)
    # fp32 products and sum (3 roundings of at most 2 |x|), then the type's
    assert ((q.double() - want).abs() <= 2.0 ** -8 * 1.01 * want.abs() + 6 * 2.0 ** -24 * x.abs().max()).all()
    if cache == "fp4":
        assert torch.equal(ops.kv4_read(kc, slots, dt).double(),
                           oracle.nearest(oracle.rotate(x[:, nq:nq + nkv], cos, sin), dt)[0])
    else:
        one = torch.stack([table[p.clamp(0, 59)] for p in pos])                # each axis alone, as one position
        for a, n in enumerate(sections):
            k2, v2 = _caches(cache, 3, nkv, bs, d, dt)
            q2 = ops.rope_kv_write(qkv, torch.arange(T), one[a].contiguous(), k2, v2, slots, nq, nkv, d)
            i = torch.arange(sum(sections[:a]), sum(sections[:a + 1]))
            i = torch.cat([i, i + d // 2])
            assert torch.equal(q[..., i], q2[..., i])
            assert torch.equal(kc.float()[..., i], k2.float()[..., i]) and torch.equal(vc.float(), v2.float())


def _caches(kind, nb, nkv, bs, d, dt):
    if kind == "fp4":
        return tuple(torch.zeros(ops.kv4_cache_shape(nb, nkv, bs, d), dtype=torch.uint8) for _ in range(2))
    t = torch.float8_e4m3fn if kind == "fp8" else dt
    return torch.zeros(nb, nkv, bs, d).to(t), torch.zeros(nb, nkv, bs // 8, d, 8).to(t)


def test_attention_reference():
    g = _gen(3)
    dt, d, nq, nkv, bs = torch.bfloat16, 64, 4, 2, 16
    new, old = [5, 1, 33], [0, 20, 7]
    totals = [a + b for a, b in zip(new, old)]
    bt, nb = oracle.tables(g, totals, bs)
    kc, vc = (oracle.random_cache(g, nb, nkv, bs, d, dt) for _ in range(2))
    q = torch.randn(sum(new), nq, d, generator=g).to(dt)
    starts = torch.tensor([0, 5, 6, 39], dtype=torch.int32)
    out = ops.prefill_attention(q, kc, vc, bt, starts, torch.tensor(totals, dtype=torch.int32), 0.125)
    last = ops.paged_attention_decode(q[starts[1:].long() - 1], kc, vc, bt, torch.tensor(totals), 0.125)
    for i, n in enumerate(totals):
        seen = torch.arange(n)[None] <= torch.arange(old[i], n)[:, None]
        for h in range(nq):
            k, v = (oracle.rows(c, bt[i], n, h // 2, d) for c in (kc, vc))
            o, tol = oracle.attend(q[starts[i]:starts[i + 1], h], k, v, 0.125, seen, dt)
            assert ((out[starts[i]:starts[i + 1], h].double() - o).abs() <= tol).all()
            assert ((last[i, h].double() - o[-1]).abs() <= tol[-1]).all()


def test_engine_with_a_4bit_cache():
    """The engine's chunked prompts and decode steps over a 4-bit cache: prompts in one chunk and in many
    write and read the same bytes, so that greedy tokens are the same."""
    from kubernetes_gpu_cluster_amd.engine.llm_engine import LLM
    from kubernetes_gpu_cluster_amd.engine.sequence import SamplingParams
    prompts = [[5 + i, 6, 7, 8, 9, 10, 11] * 5 for i in range(3)]
    sp = SamplingParams(temperature=0, max_tokens=8, ignore_eos=True)
    got = []
    for budget, kvd in ((256, "fp4"), (16, "fp4_e2m1"), (256, "auto")):
        llm = LLM("tiny-llama", device="cpu", dtype="float32", random_init=True, seed=1, max_model_len=128,
                  max_num_seqs=4, max_num_batched_tokens=budget, num_gpu_blocks_override=64, block_size=16,
                  kv_cache_dtype=kvd)
        r = llm.engine.executor.runner
        bytes_ = r.kv_bytes_per_block()
        if kvd != "auto":
            assert r.kv.dtype == torch.uint8 and r.kv.numel() == 64 * bytes_ and r.kv.any() == False  # noqa: E712
        got.append(([o.output_token_ids for o in llm.generate(prompts, sp)], bytes_))
        llm.shutdown()
    assert got[0][0] == got[1][0]
    assert got[0][1] * 128 == got[2][1] * 17                                   # 4.25 bits of 32


@pytest.mark.parametrize("model,kw,what", [
    ("tiny-dilavik", {}, "caches of its own"),
    ("tiny-llama", dict(block_size=24), "power of two"),
    ("tiny-opt", {}, "heads of 64 or 128"),
])
def test_engine_refusals(model, kw, what):
    from kubernetes_gpu_cluster_amd.engine.llm_engine import LLM
    with pytest.raises(ValueError, match=what):
        LLM(model, device="cpu", dtype="float32", random_init=True, max_model_len=128, max_num_seqs=2,
            num_gpu_blocks_override=64, kv_cache_dtype="fp4", **kw)


def test_shape_refusals():
    with pytest.raises(ValueError, match="head_dim"):
        ops.kv4_cache_shape(4, 2, 16, 96)
    from kubernetes_gpu_cluster_amd.engine.config import EngineConfig
    assert EngineConfig(kv_cache_dtype="fp4").kv_torch_dtype(torch.bfloat16) == torch.uint8


def test_decode_slices_of_a_4bit_cache():
    for B in (1, 3, 64, 256):
        for nkv in (1, 8, 12):
            for ctx in (1, 31, 640, 8192, 131072):
                z = ops.decode_grid_z(B, nkv, ctx, cache_dtype=torch.uint8)
                assert 1 <= z <= 1024 and (z == 1 or (z - 1) * 64 < ctx)
                ws = ops.decode_partials(B, nkv, 64, -(-ctx // 32), 32, "meta")
                assert z <= ws[0].numel() // (B * nkv), (B, nkv, ctx, z)


def test_slices_of_prompts_without_heads():
    """Shapes that the op refuses get there: the host's rule does not divide by their heads."""
    assert ops.kv4_prefill_slices(5, 1, 4, 0, 64, 5000) >= 1 and ops.kv4_prefill_slices(5, 1, 0, 0, 64, 5000) >= 1


@pytest.mark.parametrize("dt", DT)
def test_keys_beside_borders(dt):
    """The code is the one of the exact sum of the two products, not of its nearest 64-bit number."""
    x, table, want, e = oracle.keys_beside_borders()
    assert want[0, 5] == 3.0 and want[0, 12] == 2.0 and e[1, 0] == 1 and e[2, 0] == 0
    T = len(x)
    qkv = torch.zeros(T, 3, 64)
    qkv[:, 1] = x
    kc, vc = (torch.zeros(ops.kv4_cache_shape(1, 1, 16, 64), dtype=torch.uint8) for _ in range(2))
    slots = torch.arange(T)
    ops.rope_kv_write(qkv.to(dt).view(T, -1), slots * 0, table, kc, vc, slots, 1, 1, 64)
    assert torch.equal(ops.kv4_read(kc, slots, dt)[:, 0].double(), want)
    assert torch.equal(ref.kv4_parts(kc)[1][0, 0, :T].double() - 127, e)


def test_cpu_forms_refuse_what_the_kernels_refuse():
    d, T = 64, 3
    kc, vc = (torch.zeros(ops.kv4_cache_shape(2, 1, 16, d), dtype=torch.uint8) for _ in range(2))
    table, x, slots = torch.ones(8, d), torch.ones(T, 4 * d, dtype=torch.bfloat16), torch.arange(T)
    two = torch.zeros(2, T, dtype=torch.int64)

    def no(what, f, *a, **k):
        with pytest.raises(ValueError, match=what):
            f(*a, **k)

    def write(pos, table=table, **k):
        return ops.rope_kv_write(x, pos, table, kc, vc, slots, 2, 1, d, **k)
    no("own scales", write, slots, k_scale=0.5)
    no("sections of a rotated head", write, two, sections=(16, 16), use_rope=False)
    no("1 to 4", write, torch.zeros(5, T, dtype=torch.int64), sections=(28, 1, 1, 1, 1))
    no("1 to 4", write, torch.zeros(0, T, dtype=torch.int64), sections=())
    no("all of them 32", write, two, sections=(16, 15))
    no("0 to d / 2", write, two, sections=(-1, 33))
    no(r"\[sections, T\]", write, slots, sections=(16, 16))
    no(r"\[sections, T\]", write, two[:, :2], sections=(16, 16))
    no("empty cos_sin", write, two, table[:0], sections=(16, 16))
    assert not kc.any() and not vc.any()
    q, bt, n = torch.ones(1, 2, d, dtype=torch.bfloat16), torch.zeros(1, 1, dtype=torch.int32), torch.tensor([2])
    no("own scales", ops.paged_attention_decode, q, kc, vc, bt, n, 1.0, v_scale=2.0)
    no("own scales", ops.prefill_attention, q, kc, vc, bt, torch.tensor([0, 1]), n, 1.0, k_scale=2.0)
