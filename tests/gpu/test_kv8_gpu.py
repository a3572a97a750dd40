"""The kernels of the 8-bit cache and of norm + rotation against a 64-bit
oracle, at the sizes, strides and masks where they could go wrong."""

import pytest
import torch

from tests import kv8_oracle as oracle

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from fma_amd.ops import actuation, decode_ops, kv8
    actuation.require_native()
    kv8.fast_qk_norm_rope = decode_ops.fast_qk_norm_rope
    return kv8


def randn(*shape, dtype=BF, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def value(x, dtype):
    return x.float().to(dtype)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def filled(ops, n, H=2, hd=128, B=1, fmt="fp8", dtype=BF, cap=None, seed=0,
           kscale=2.0):
    """A cache of n tokens and the raw keys and values in it."""
    c = ops.KV8Cache(2, B, cap or n, H, hd, fmt=fmt, dtype=dtype,
                     device="cuda")
    k = randn(B, n, H, hd, dtype=dtype, seed=seed, scale=kscale)
    v = randn(B, n, H, hd, dtype=dtype, seed=seed + 1)
    ops.kv8_append(c, 1, k, v, 0)
    return c, k, v


# -- norm and rotation ---------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("hd,rot", [(128, 128), (128, 64), (64, 64), (80, 30),
                                    (96, 96), (256, 256), (2, 2), (33, 20),
                                    (160, 158)])
@pytest.mark.parametrize("norm", [True, False])
def test_norm_rope(ops, dtype, interleaved, hd, rot, norm):
    q = randn(3, 7, 5, hd, dtype=dtype, scale=3.0)
    k = randn(3, 7, 2, hd, dtype=dtype, seed=1)
    cos, sin = oracle.tables(100, rot, "cuda", factor=1.1)
    w = [randn(hd, dtype=dtype, seed=s) if norm else None for s in (2, 3)]
    pos = torch.randint(0, 100, (3, 7), device="cuda")
    got = ops.fast_qk_norm_rope(q, k, cos, sin, pos, *w, eps=1e-5,
                                interleaved=interleaved)
    for x, y, g in zip((q, k), got, w):
        assert y.shape == x.shape and y.is_contiguous()
        want, bound = oracle.norm_rope(x, g, cos, sin, pos, 1e-5, interleaved)
        oracle.check(y, want, bound, dtype)


@pytest.mark.parametrize("B,T,qh,kvh", [(1, 1, 32, 8), (1, 1000, 32, 8),
                                        (2, 301, 9, 3), (64, 1, 64, 8),
                                        (1, 2, 1, 1), (1, 4097, 7, 1)])
def test_norm_rope_sizes(ops, B, T, qh, kvh):
    q, k = randn(B, T, qh, 128), randn(B, T, kvh, 128, seed=1)
    cos, sin = oracle.tables(5000, 128, "cuda")
    w = randn(128, seed=4)
    got = ops.fast_qk_norm_rope(q, k, cos, sin, 17, w, None)
    pos = (17 + torch.arange(T)).expand(B, T)
    for x, y, g in zip((q, k), got, (w, None)):
        want, bound = oracle.norm_rope(x, g, cos, sin, pos, 1e-6, True)
        oracle.check(y, want, bound, BF)


def test_norm_rope_strides_positions_and_outside(ops):
    cos, sin = oracle.tables(50, 64, "cuda")
    qkv = randn(2, 6, 10, 64)
    odd = randn(2, 6, 10, 65)[..., 1:]            # rows on odd addresses
    swapped = randn(6, 10, 2, 64).permute(2, 0, 1, 3)
    last = randn(2, 64, 6, 10).permute(0, 2, 3, 1)
    for x in (qkv, odd, swapped, last):
        a = ops.fast_qk_norm_rope(x[:, :, :7], x[:, :, 7:], cos, sin, 3)
        b = ops.fast_qk_norm_rope(x[:, :, :7].contiguous(),
                                  x[:, :, 7:].contiguous(), cos, sin,
                                  ints(3, 3))
        c = ops.fast_qk_norm_rope(
            x[:, :, :7], x[:, :, 7:], cos, sin,
            (3 + torch.arange(6, device="cuda")).expand(2, 6))
        for u, w, z in zip(a, b, c):
            assert torch.equal(u, w) and torch.equal(u, z)
    a = ops.fast_qk_norm_rope(qkv[:, :, :7], qkv[:, :, 7:], cos, sin,
                              ints(46, -1))
    assert torch.isnan(a[0][0, 4:]).all() and torch.isnan(a[1][1, 0]).all()
    assert torch.isfinite(a[0][0, :4]).all()
    assert torch.isfinite(a[1][1, 1:]).all()


def test_norm_rope_extreme_rows(ops):
    """Zeros, and rows whose squares sum to near fp32's ends."""
    cos, sin = oracle.tables(8, 64, "cuda")
    q = randn(1, 3, 1, 64, dtype=BF)
    q[0, 0] = 0
    q[0, 1] *= 1e18
    q[0, 2] *= 1e-12
    w = torch.ones(64, device="cuda", dtype=BF)
    got, _ = ops.fast_qk_norm_rope(q, q, cos, sin, 0, w, w)
    want, bound = oracle.norm_rope(q, w, cos, sin, torch.arange(3)[None],
                                   1e-6, True)
    oracle.check(got, want, bound, BF)


# -- store and read back -------------------------------------------------------

@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hd", [16, 33, 64, 80, 96, 128, 160, 256])
@pytest.mark.parametrize("n", [1, 31, 32, 33, 200])
def test_read_gives_what_the_definition_says(ops, fmt, dtype, hd, n):
    c, k, v = filled(ops, n, hd=hd, B=2, fmt=fmt, dtype=dtype)
    rk, rv = ops.kv8_read(c, 1, 0, n + 5, n)
    for b in range(2):
        assert torch.equal(rk[b, :n].cpu(),
                           value(oracle.held(k[b], fmt), dtype))
        assert torch.equal(rv[b, :n].cpu(),
                           value(oracle.held(v[b], fmt), dtype))
    assert not rk[:, n:].any() and not rv[:, n:].any()
    assert not c.codes[0].any() and not c.tail[0].any()  # the other layer


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_result_does_not_depend_on_how_tokens_arrive(ops, fmt):
    H, n = 3, 201
    whole, k, v = filled(ops, n, H=H, fmt=fmt)
    parts = ops.KV8Cache(1, 1, 256, H, 128, fmt=fmt, device="cuda")
    at = 0
    for m in (1, 30, 1, 5, 40, 3, 17, 70, 34):
        ops.kv8_append(parts, 0, k[:, at:at + m], v[:, at:at + m], at)
        at += m
        got = ops.kv8_read(parts, 0, 0, at, at)
        for x, y in zip(got, (k, v)):
            assert torch.equal(x[0].cpu(), value(
                oracle.held(y[0, :at], fmt), BF))
    assert at == n


def test_store_on_the_cpu_lies_the_same(ops):
    for fmt in ("fp8", "int8"):
        c, k, v = filled(ops, 75, hd=80, fmt=fmt)
        cpu = ops.KV8Cache(2, 1, 75, 2, 80, fmt=fmt)
        ops.kv8_append(cpu, 1, k.cpu(), v.cpu(), 0)
        assert torch.equal(c.scales.cpu(), cpu.scales)
        got, want = (ops.kv8_read(x, 1, 0, 75, 75) for x in (c, cpu))
        for a, b in zip(got, want):
            assert torch.equal(a.cpu(), b)
        assert torch.equal(c.codes[1, :, :, :, :2].cpu(),
                           cpu.codes[1, :, :, :, :2])


def test_going_back_and_slots(ops):
    c, k, v = filled(ops, 62, H=8, cap=300)
    ops.kv8_append(c, 1, *(randn(1, 5, 8, 128, seed=s) for s in (8, 9)), 62)
    k2, v2 = randn(1, 98, 8, 128, seed=3), randn(1, 98, 8, 128, seed=4)
    ops.kv8_append(c, 1, k2, v2, 62)     # reads slot 1, ends in slot 1
    for x, y, z in zip(ops.kv8_read(c, 1, 0, 160, 160), (k, v), (k2, v2)):
        raw = torch.cat((y[0], z[0]))
        assert torch.equal(x[0].cpu(), value(oracle.held(raw, "fp8"), BF))
    for end in (70, 96, 97, 130, 161, 162):
        k3, v3 = randn(1, end, 8, 128, seed=5), randn(1, end, 8, 128, seed=6)
        d = ops.KV8Cache(1, 1, 200, 8, 128, fmt="int8", device="cuda")
        ops.kv8_append(d, 0, k3[:, :5], v3[:, :5], 0)
        ops.kv8_append(d, 0, k3[:, 5:], v3[:, 5:], 5)
        for x, y in zip(ops.kv8_read(d, 0, 0, end, end), (k3, v3)):
            assert torch.equal(x[0].cpu(),
                               value(oracle.held(y[0], "int8"), BF))


def test_ragged_store_leaves_the_rest(ops):
    """Starts and counts from the GPU, a slot without tokens, padding with
    NaN, a sequence that would pass the end, and starts outside."""
    B, H, T = 6, 2, 70
    c = ops.KV8Cache(1, B, 128, H, 128, device="cuda")
    before = [x.clone() for x in (c.codes, c.scales, c.tail)]
    start = ints(0, 32, 64, 96, -1, 129)
    counts = ints(70, 0, 40, 70, 5, 5)
    k, v = randn(B, T, H, 128), randn(B, T, H, 128, seed=1)
    k[2, 40:], v[2, 40:] = float("nan"), float("nan")
    ops.kv8_append(c, 0, k, v, start, counts)
    for b, s, n in ((0, 0, 70), (2, 64, 40), (3, 96, 32)):
        lo, end = ints(*[s] * B), ints(*[s + n] * B)
        for x, y in zip(ops.kv8_read(c, 0, lo, T, end), (k, v)):
            assert torch.equal(x[b, :n].cpu(),
                               value(oracle.held(y[b, :n], "fp8"), BF))
            assert not x[b, n:].any()
    for b in (1, 4, 5):
        for x, y in zip((c.codes, c.scales, c.tail), before):
            assert torch.equal(x[:, :, b], y[:, :, b])
    # blocks in front of and behind a sequence's tokens
    assert not c.codes[:, :, 2, :, :2].any()
    assert not c.codes[:, :, 2, :, 3:].any()
    assert not c.codes[:, :, 3, :, :3].any()


def test_not_finite_values(ops):
    for fmt in ("fp8", "int8"):
        k, v = randn(1, 40, 2, 128), randn(1, 40, 2, 128, seed=1)
        k[0, 3, 0, 1], k[0, 4, 1, 2] = float("nan"), float("inf")
        v[0, 5, 0, 0], v[0, 6] = float("-inf"), float("nan")
        v[0, :32, 1] = float("inf")
        c = ops.KV8Cache(1, 1, 64, 2, 128, fmt=fmt, device="cuda")
        ops.kv8_append(c, 0, k, v, 0)
        for x, y in zip(ops.kv8_read(c, 0, 0, 32, 40), (k, v)):
            assert torch.equal(x[0].cpu(),
                               value(oracle.held(y[0, :32], fmt), BF))


def test_scales_at_the_ends_of_the_types(ops):
    """Zeros, magnitudes under 2^-100, near bf16's largest, and the steps
    where the fp8 scale changes."""
    for fmt in ("fp8", "int8"):
        for top in (0.0, 2.0 ** -120, 2.0 ** -100, 3e38, 448.0, 450.0, 1.75,
                    1.7578125, 1.0, 2.0):
            k = torch.full((1, 32, 1, 64), top / 3, device="cuda", dtype=BF)
            k[0, 7, 0, 9] = top
            c = ops.KV8Cache(1, 1, 32, 1, 64, fmt=fmt, device="cuda")
            ops.kv8_append(c, 0, k, -k, 0)
            rk, rv = ops.kv8_read(c, 0, 0, 32, 32)
            assert torch.equal(rk[0].cpu(), value(oracle.held(k[0], fmt), BF))
            assert torch.equal(rv, -rk)
    # a code may stand for more than the type holds: it saturates
    for dtype in (BF, HF):
        k = torch.full((1, 32, 1, 64), torch.finfo(dtype).max, device="cuda",
                       dtype=dtype)
        c = ops.KV8Cache(1, 1, 32, 1, 64, dtype=dtype, device="cuda")
        d = ops.KV8Cache(1, 1, 32, 1, 64, dtype=dtype)
        ops.kv8_append(c, 0, k, -k, 0)
        ops.kv8_append(d, 0, k.cpu(), -k.cpu(), 0)
        rk, rv = ops.kv8_read(c, 0, 0, 32, 32)
        assert torch.equal(rk, k) and torch.equal(rv, -k)
        assert torch.equal(ops.kv8_read(d, 0, 0, 32, 32)[0], k.cpu())


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("hd,rot,norm", [(128, 128, True), (64, 64, False),
                                         (80, 20, True), (256, 256, True)])
@pytest.mark.parametrize("start,T", [(0, 1), (31, 1), (0, 100), (37, 60)])
def test_one_call_is_the_two_calls(ops, interleaved, hd, rot, norm, start, T):
    B, H = 2, 2
    q, k, v = (randn(B, T, n, hd, seed=s) for n, s in ((6, 0), (H, 1), (H, 2)))
    cos, sin = oracle.tables(160, rot, "cuda")
    w = randn(hd, seed=5) if norm else None
    a, b = (ops.KV8Cache(1, B, 160, H, hd, device="cuda") for _ in range(2))
    if start:
        old = randn(B, start, H, hd, seed=7)
        for c in (a, b):
            ops.kv8_append(c, 0, old, old, 0)
    qa = ops.qk_norm_rope_kv8(a, 0, q, k, v, cos, sin, start, w, w,
                              interleaved=interleaved)
    qb, kb = ops.fast_qk_norm_rope(q, k, cos, sin, start, w, w,
                                   interleaved=interleaved)
    ops.kv8_append(b, 0, kb, v, start)
    assert torch.equal(qa, qb)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    assert torch.equal(a.tail, b.tail)
    counts = ints(T, 0)
    qc = ops.qk_norm_rope_kv8(a, 0, q, k, v, cos, sin, ints(start, start), w,
                              w, counts=counts, interleaved=interleaved)
    assert torch.equal(qc[0], qb[0]) and not qc[1].any()


# -- attention -----------------------------------------------------------------

def attend_and_check(ops, c, q, k, v, start, scale=None):
    fmt, dtype = c.fmt, q.dtype
    T = q.shape[1]
    out = ops.kv8_attention(q, c, 1, start, scale=scale)
    for b in range(q.shape[0]):
        n = start + T
        want, bound = oracle.attention(
            q[b], oracle.held(k[b, :n], fmt), oracle.held(v[b, :n], fmt),
            start, q.shape[3] ** -0.5 if scale is None else scale)
        oracle.check(out[b], want, bound, dtype)
    return out


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hd", [16, 33, 64, 80, 96, 128, 160, 256])
@pytest.mark.parametrize("n", [1, 32, 75, 300])
def test_attention_token(ops, fmt, dtype, hd, n):
    c, k, v = filled(ops, n, hd=hd, B=2, fmt=fmt, dtype=dtype)
    q = randn(2, 1, 8, hd, dtype=dtype, seed=2)
    attend_and_check(ops, c, q, k, v, n - 1)


@pytest.mark.parametrize("qh,kvh", [(1, 1), (7, 1), (16, 1), (20, 1), (64, 2),
                                    (28, 4)])
@pytest.mark.parametrize("n", [31, 64, 1000, 5000])
def test_attention_groups_and_lengths(ops, qh, kvh, n):
    c, k, v = filled(ops, n, H=kvh)
    q = randn(1, 1, qh, 128, seed=2)
    attend_and_check(ops, c, q, k, v, n - 1)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
@pytest.mark.parametrize("start,T", [(0, 2), (0, 33), (30, 5), (64, 64),
                                     (100, 129), (1, 300), (700, 17)])
def test_attention_chunk(ops, fmt, hd, start, T):
    n = start + T
    c, k, v = filled(ops, n, hd=hd, fmt=fmt, dtype=HF if hd == 96 else BF)
    q = randn(1, T, 12, hd, dtype=k.dtype, seed=2)
    attend_and_check(ops, c, q, k, v, start)


@pytest.mark.parametrize("qh,kvh", [(1, 1), (3, 1), (16, 1), (17, 1), (40, 8)])
def test_attention_chunk_groups(ops, qh, kvh):
    c, k, v = filled(ops, 450, H=kvh)
    q = randn(1, 250, qh, 128, seed=2)
    attend_and_check(ops, c, q, k, v, 200)


def test_attention_peaked_and_uneven(ops):
    """Rows that one far token holds, first or last; V blocks of very
    different scale; a scale argument; queries of tiny and huge size."""
    for fmt in ("fp8", "int8"):
        c, k, v = filled(ops, 400, fmt=fmt, cap=1000)
        for big in (0, 399):
            kk, vv = k.clone(), v.clone()
            kk[:, big] *= 20
            vv[:, :64] *= 1e-3
            vv[:, 64:160] *= 300
            vv[:, 320:] *= 1e-6
            ops.kv8_append(c, 1, kk, vv, 0)
            q = randn(1, 3, 8, 128, seed=2)
            q[:, :, 1] = kk[0, big, 0]
            q[:, :, 2] *= 1e-6
            q[:, :, 3] *= 1e6
            q[:, :, 4] = 0
            q[:, :, 5, 1:] *= 1e-7
            attend_and_check(ops, c, q, kk, vv, 397)
            attend_and_check(ops, c, q[:, :, :2], kk, vv, 397, scale=1.0)
            attend_and_check(ops, c, q[:, :, :2], kk, vv, 397, scale=-0.2)


def test_attention_ignores_what_is_masked(ops):
    """NaN and infinities behind the last token, in padding, in later tokens
    of the same call and in other sequences reach no row that cannot see
    them."""
    for fmt in ("fp8", "int8"):
        for T in (3, 90):
            B, H, n = 3, 2, 100
            c = ops.KV8Cache(2, B, 256, H, 128, fmt=fmt, device="cuda")
            c.tail.fill_(float("nan"))
            c.codes.fill_(0x7f)
            c.scales.fill_(float("nan"))
            k, v = randn(B, n, H, 128), randn(B, n, H, 128, seed=1)
            start = ints(n - T, n - T, n - T)
            counts = ints(T, 0, T - 1)
            ops.kv8_append(c, 1, k[:, :n - T], v[:, :n - T], 0,
                           counts=ints(n - T, 0, n - T))
            kk, vv = k.clone(), v.clone()
            kk[2, n - 1] = float("nan")          # padding
            kk[0, n - 1], vv[0, n - 1] = float("inf"), float("nan")
            ops.kv8_append(c, 1, kk[:, n - T:], vv[:, n - T:], start, counts)
            q = randn(B, T, 8, 128, seed=4)
            q[1] = float("nan")
            out = ops.kv8_attention(q, c, 1, start, counts)
            assert not out[1].any() and not out[2, T - 1:].any()
            for b, live in ((0, T - 1), (2, T - 1)):
                m = n - 1
                # what is coded lies in front of token 96
                want, bound = oracle.attention(
                    q[b, :live], oracle.held(k[b, :m], fmt),
                    oracle.held(v[b, :m], fmt), n - T, 128 ** -0.5)
                oracle.check(out[b, :live], want, bound, BF)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("T", [2, 40, 150])
def test_attention_over_blocks_of_uneven_scale(ops, fmt, T):
    """V's scale up and down by up to 2^40 from one block to the next, and
    blocks of zeros, for few rows and for many."""
    n = 500
    k, v = randn(1, n, 2, 128), randn(1, n, 2, 128, seed=1)
    for i, e in enumerate((0, 7, -7, 0, 20, 0, -13, -40, 0, 3, 9, -9, 6, -6,
                           12, 0)):
        v[:, 32 * i:32 * i + 32] *= 2.0 ** e
    v[:, 160:192], k[:, 224:288] = 0, 0
    c = ops.KV8Cache(2, 1, n, 2, 128, fmt=fmt, device="cuda")
    ops.kv8_append(c, 1, k, v, 0)
    q = randn(1, T, 8, 128, seed=2)
    q[:, :, 3] *= 30                          # one block holds the row
    attend_and_check(ops, c, q, k, v, n - T)


@pytest.mark.parametrize("T,qh,kvh,n,B", [(200, 16, 1, 3300, 1),
                                          (70, 12, 2, 4000, 1),
                                          (1, 64, 2, 700, 32),
                                          (12, 8, 2, 3000, 2)])
def test_attention_splits_and_joins(ops, T, qh, kvh, n, B):
    c, k, v = filled(ops, n, H=kvh, B=B, hd=64)
    q = randn(B, T, qh, 64, seed=2)
    attend_and_check(ops, c, q, k, v, n - T)


def test_attention_scale_zero_is_the_mean(ops):
    c, k, v = filled(ops, 100)
    q = randn(1, 30, 8, 128, seed=2)
    attend_and_check(ops, c, q, k, v, 70, scale=0.0)


def test_queries_in_front_of_the_last_token(ops):
    c, k, v = filled(ops, 150)
    for start, T in ((49, 1), (40, 30), (0, 3), (127, 2), (95, 1), (20, 90)):
        q = randn(1, T, 8, 128, seed=2)
        out = ops.kv8_attention(q, c, 1, start)
        n = start + T
        want, bound = oracle.attention(
            q[0], oracle.held(k[0], "fp8")[:n], oracle.held(v[0], "fp8")[:n],
            start, 128 ** -0.5)
        oracle.check(out[0], want, bound, BF)


def test_capacity_inside_a_block(ops):
    """max_seq 45: the last token, and tokens dropped behind it."""
    c = ops.KV8Cache(2, 1, 45, 2, 128, device="cuda")
    k, v = randn(1, 45, 2, 128), randn(1, 45, 2, 128, seed=1)
    ops.kv8_append(c, 1, k, v, 0)
    q = randn(1, 45, 8, 128, seed=2)
    attend_and_check(ops, c, q, k, v, 0)
    d = ops.KV8Cache(1, 1, 45, 2, 128, device="cuda")
    wide = torch.cat((k, k), 1)
    ops.kv8_append(d, 0, wide, torch.cat((v, v), 1), ints(0))
    assert torch.equal(d.codes[0], c.codes[1])
    for x, y in zip(ops.kv8_read(d, 0, 0, 45, ints(45)), (k, v)):
        assert torch.equal(x[0].cpu(), value(oracle.held(y[0], "fp8"), BF))
    out = ops.kv8_attention(randn(1, 90, 8, 128), d, 0, ints(0))
    assert not out[:, 45:].any()


def test_read_from_inside_a_block(ops):
    c, k, v = filled(ops, 150, B=2)
    for x, y in zip(ops.kv8_read(c, 1, 5, 100, 150), (k, v)):
        assert torch.equal(x[1].cpu(), value(
            oracle.held(y[1], "fp8")[5:105], BF))
    got = ops.kv8_read(c, 1, ints(140, 3), 20, ints(150, 150))
    for x, y in zip(got, (k, v)):
        h = oracle.held(y[0], "fp8")
        assert torch.equal(x[0, :10].cpu(), value(h[140:], BF))
        assert not x[0, 10:].any()
        h = oracle.held(y[1], "fp8")
        assert torch.equal(x[1].cpu(), value(h[3:23], BF))


def test_large_outputs_have_the_same_bits(ops):
    """Outputs beyond the caches are stored past them."""
    T = 5000
    q, k, v = randn(1, T, 32, 128), randn(1, T, 8, 128), randn(1, T, 8, 128)
    cos, sin = oracle.tables(T, 128, "cuda")
    w = randn(128, seed=3)
    got = ops.fast_qk_norm_rope(q, k, cos, sin, 0, w, w)
    c, d = (ops.KV8Cache(1, 1, T, 8, 128, device="cuda") for _ in range(2))
    qc = ops.qk_norm_rope_kv8(c, 0, q, k, v, cos, sin, 0, w, w)
    assert torch.equal(qc, got[0])
    for at in range(0, T, 800):
        s = slice(at, at + 800)
        part = ops.fast_qk_norm_rope(q[:, s], k[:, s], cos, sin, at, w, w)
        assert torch.equal(part[0], got[0][:, s])
        assert torch.equal(part[1], got[1][:, s])
        ops.qk_norm_rope_kv8(d, 0, q[:, s], k[:, s], v[:, s], cos, sin, at, w,
                             w)
    assert torch.equal(c.codes, d.codes) and torch.equal(c.scales, d.scales)


def test_refusals_on_the_gpu(ops):
    """The same as on the CPU; nothing is launched."""
    c, k, v = filled(ops, 10, cap=100)
    cos, sin = oracle.tables(100, 128, "cuda")
    q = randn(1, 1, 8, 128)
    w = torch.ones(128, device="cuda", dtype=BF)
    bad = [
        lambda: ops.kv8_append(c, 2, k, v, 10),
        lambda: ops.kv8_append(c, 1, k[..., :64], v, 10),
        lambda: ops.kv8_append(c, 1, k.float(), v, 10),
        lambda: ops.kv8_append(c, 1, k.cpu(), v, 10),
        lambda: ops.kv8_append(c, 1, k, v[:, :5], 10),
        lambda: ops.kv8_append(c, 1, k[:, :, :1], v[:, :, :1], 10),
        lambda: ops.kv8_append(c, 1, k, v, 95),
        lambda: ops.kv8_append(c, 1, k, v, -1),
        lambda: ops.kv8_append(c, 1, k, v, 12),
        lambda: ops.kv8_append(c, 1, k, v, ints(0, 0)),
        lambda: ops.kv8_append(c, 1, k, v, torch.tensor([0], device="cuda")),
        lambda: ops.kv8_append(c, 1, k, v, ints(0).cpu()),
        lambda: ops.kv8_append(c, 1, k, v, 10, ints(1, 2)),
        lambda: ops.kv8_append(c, 1, k.clone().requires_grad_(), v, 10),
        lambda: ops.kv8_attention(q, c, 1, 10),
        lambda: ops.kv8_attention(q[:, :, :3], c, 1, 9),
        lambda: ops.kv8_attention(q.half(), c, 1, 9),
        lambda: ops.kv8_attention(q.cpu(), c, 1, 9),
        lambda: ops.kv8_attention(q[0], c, 1, 9),
        lambda: ops.kv8_read(c, 1, 0, 5, 11),
        lambda: ops.kv8_read(c, 1, 0, -1, 10),
        lambda: ops.qk_norm_rope_kv8(c, 1, q, k, v, cos, sin, 10),
        lambda: ops.qk_norm_rope_kv8(c, 1, q, k[:, :1], v[:, :1], cos[:99],
                                     sin[:99], 10),
        lambda: ops.fast_qk_norm_rope(q, q, cos, sin, 100),
        lambda: ops.fast_qk_norm_rope(q, q, cos, sin[:50], 0),
        lambda: ops.fast_qk_norm_rope(q, q, cos.half(), sin.half(), 0),
        lambda: ops.fast_qk_norm_rope(q, q, cos, sin, 0, w[:64]),
        lambda: ops.fast_qk_norm_rope(q, q, cos, sin, 0, w.float()),
        lambda: ops.fast_qk_norm_rope(q, q, cos, sin, ints(0, 1)),
        lambda: ops.fast_qk_norm_rope(q, q.half(), cos, sin, 0),
        lambda: ops.fast_qk_norm_rope(q, k, cos, sin, 0),
        lambda: ops.fast_qk_norm_rope(q.clone().requires_grad_(), q, cos, sin,
                                      0),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    # the refused calls have changed nothing
    ops.kv8_append(c, 1, k, v, 10)
    assert torch.equal(ops.kv8_read(c, 1, 10, 10, 20)[0], k)


def test_attention_nan_query_stays_in_its_row(ops):
    c, k, v = filled(ops, 90)
    q = randn(1, 20, 8, 128, seed=2)
    clean = ops.kv8_attention(q, c, 1, 70)
    q[0, 3, 5] = float("nan")
    out = ops.kv8_attention(q, c, 1, 70)
    assert torch.isnan(out[0, 3, 5]).all()
    out[0, 3, 5] = clean[0, 3, 5]
    assert torch.equal(out, clean)


def test_attention_ragged_on_the_gpu(ops):
    B, H, T = 9, 2, 4
    k, v = randn(B, 600, H, 64), randn(B, 600, H, 64, seed=1)
    c = ops.KV8Cache(2, B, 640, H, 64, device="cuda")
    ends = [4, 5, 33, 600, 1, 100, 32, 64, 599]
    ops.kv8_append(c, 1, k, v, 0, counts=ints(*ends))
    counts = [4, 0, 3, 4, 1, 2, 4, 1, 4]
    start = [e - n for e, n in zip(ends, counts)]
    q = randn(B, T, 6, 64, seed=3)
    out = ops.kv8_attention(q, c, 1, ints(*start), ints(*counts))
    for b in range(B):
        n = counts[b]
        assert not out[b, n:].any()
        if n:
            want, bound = oracle.attention(
                q[b, :n], oracle.held(k[b, :ends[b]], "fp8"),
                oracle.held(v[b, :ends[b]], "fp8"), start[b], 0.125)
            oracle.check(out[b, :n], want, bound, BF)
    # positions outside the cache: nothing, and nothing read
    out = ops.kv8_attention(q, c, 1, ints(*[-1, 641] + [640] * (B - 2)))
    assert not out.any()


def test_attention_strides(ops):
    c, k, v = filled(ops, 130)
    q = randn(1, 3, 8, 128, seed=2)
    want = ops.kv8_attention(q, c, 1, 127)
    wide = randn(1, 3, 24, 128)
    wide[:, :, 3:11] = q
    odd = torch.zeros(1, 3, 8, 129, device="cuda", dtype=BF)[..., 1:]
    odd.copy_(q)
    last = q.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)
    for x in (wide[:, :, 3:11], odd, last):
        assert torch.equal(ops.kv8_attention(x, c, 1, 127), want)


def test_empty_calls(ops):
    c, k, v = filled(ops, 40, cap=64)
    q = randn(1, 0, 8, 128)
    assert ops.kv8_attention(q, c, 1, 40).shape == (1, 0, 8, 128)
    ops.kv8_append(c, 1, k[:, :0], v[:, :0], 40)
    cos, sin = oracle.tables(64, 128, "cuda")
    assert ops.qk_norm_rope_kv8(c, 1, q, k[:, :0], v[:, :0], cos, sin,
                                40).numel() == 0
    assert ops.fast_qk_norm_rope(q, q, cos, sin, 0)[0].numel() == 0
    assert ops.kv8_read(c, 1, 0, 0, 40)[0].shape == (1, 0, 2, 128)


# -- together, streams and graphs ------------------------------------------------

def decode_chain(ops, c, q, k, v, cos, sin, w, start):
    q = ops.qk_norm_rope_kv8(c, 0, q, k, v, cos, sin, start, w, w)
    return ops.kv8_attention(q, c, 0, start)


def test_prompt_then_tokens(ops):
    """Prompt, then single tokens, against the oracle over all of it."""
    H, n, P = 2, 110, 75
    q, k, v = (randn(1, n, m, 64, seed=s) for m, s in ((8, 0), (H, 1), (H, 2)))
    cos, sin = oracle.tables(128, 64, "cuda")
    w = randn(64, seed=5)
    qn, kn = ops.fast_qk_norm_rope(q, k, cos, sin, 0, w, w)
    c = ops.KV8Cache(1, 1, 128, H, 64, device="cuda")
    at = 0
    for m in [P] + [1] * (n - P):
        s = slice(at, at + m)
        out = decode_chain(ops, c, q[:, s], k[:, s], v[:, s], cos, sin, w, at)
        at += m
        want, bound = oracle.attention(
            qn[0, s], oracle.held(kn[0, :at], "fp8"),
            oracle.held(v[0, :at], "fp8"), at - m, 0.125)
        oracle.check(out[0], want, bound, BF)


def test_captured_steps_replay(ops):
    """A captured step whose position advances on the GPU, replayed with
    eager work in between; two graphs of one cache's layers."""
    B, H, n = 2, 2, 100
    q, k, v = (randn(B, n, m, 64, seed=s) for m, s in ((8, 0), (H, 1), (H, 2)))
    cos, sin = oracle.tables(128, 64, "cuda")
    w = randn(64, seed=5)
    eager = ops.KV8Cache(1, B, 128, H, 64, device="cuda")
    caches = [ops.KV8Cache(1, B, 128, H, 64, device="cuda") for _ in range(2)]
    start = torch.zeros(B, dtype=torch.int32, device="cuda")
    bufs = [torch.zeros_like(x[:, :1]) for x in (q, k, v)]
    graphs, outs = [], []
    for c in caches:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            decode_chain(ops, c, *bufs, cos, sin, w, start)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(decode_chain(ops, c, *bufs, cos, sin, w, start))
        graphs.append(g)
    for t in range(n):
        for x, y in zip(bufs, (q, k, v)):
            x.copy_(y[:, t:t + 1])
        start.fill_(t)
        for g in graphs:
            g.replay()
        want = decode_chain(ops, eager, *(x[:, t:t + 1] for x in (q, k, v)),
                            cos, sin, w, start)
        for out in outs:
            assert torch.equal(out, want), t
    torch.cuda.synchronize()


def test_captured_attention_with_splits(ops):
    """Split over a long axis inside a graph: positions change under it."""
    B, H, cap = 2, 2, 4096
    c = ops.KV8Cache(1, B, cap, H, 64, device="cuda")
    k, v = randn(B, cap, H, 64), randn(B, cap, H, 64, seed=1)
    q = randn(B, 1, 8, 64, seed=2)
    start = ints(0, 0)
    ops.kv8_append(c, 0, k, v, 0, counts=start + 1)
    ops.kv8_attention(q, c, 0, start)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.kv8_attention(q, c, 0, start)
    for ends in ((1, 4096), (4000, 77), (33, 32), (2048, 3000)):
        ops.kv8_append(c, 0, k, v, 0, counts=ints(*ends))
        start.copy_(ints(*ends) - 1)
        g.replay()
        eager = ops.kv8_attention(q, c, 0, start)
        assert torch.equal(out, eager)
        for b, n in enumerate(ends):
            want, bound = oracle.attention(
                q[b], oracle.held(k[b, :n], "fp8"),
                oracle.held(v[b, :n], "fp8"), n - 1, 0.125)
            oracle.check(out[b], want, bound, BF)


def test_on_another_stream_and_twice_at_once(ops):
    c, k, v = filled(ops, 3000, H=4)
    q = randn(1, 1, 32, 128, seed=2)
    want = ops.kv8_attention(q, c, 1, 2999)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(5):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(ops.kv8_attention(q, c, 1, 2999))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_cache_beyond_32_bit_offsets(ops):
    """Codes of more than 2^32 bytes: the last sequence's blocks."""
    B, S, H, hd = 17, 1 << 20, 1, 128
    c = ops.KV8Cache(1, B, S, H, hd, device="cuda")
    assert c.codes.numel() > 1 << 32
    n = 100
    k, v = randn(B, n, H, hd), randn(B, n, H, hd, seed=1)
    lo = S - 128
    start = ints(*[lo] * B)
    ops.kv8_append(c, 0, k, v, start)
    for x, y in zip(ops.kv8_read(c, 0, lo, n, lo + n), (k, v)):
        for b in (0, B - 1):
            assert torch.equal(x[b].cpu(),
                               value(oracle.held(y[b], "fp8"), BF))
    # the zeros in front have no scale: give them one, and attend over all
    c.scales.fill_(1.0)
    ops.kv8_append(c, 0, k, v, start)
    q = randn(B, 1, 4, hd, seed=2)
    out = ops.kv8_attention(q, c, 0, ints(*[lo + n - 1] * B))
    b = B - 1
    kh = torch.cat((torch.zeros(lo, H, hd).double(), oracle.held(k[b], "fp8")))
    vh = torch.cat((torch.zeros(lo, H, hd).double(), oracle.held(v[b], "fp8")))
    want, bound = oracle.attention(q[b], kh, vh, lo + n - 1, hd ** -0.5)
    oracle.check(out[b], want, bound, BF)


# -- the framework's own paths over it -------------------------------------------

@pytest.mark.parametrize("kv", ["fp8", "int8"])
@pytest.mark.parametrize("qk_norm", [False, True])
def test_engine_over_an_8bit_cache(kv, qk_norm):
    """Prompt, graph replays and a sleep/wake cycle; the replayed steps give
    what the same steps give eagerly."""
    from fma_amd.models.decode_graph import StaticDecoder
    from fma_amd.models.llama import LlamaConfig
    from fma_amd.runtime.engine import ActuationEngine
    cfg = LlamaConfig(name="kv8", vocab_size=512, hidden_size=512,
                      intermediate_size=768, num_layers=2, num_heads=4,
                      num_kv_heads=2, max_seq_len=256, qk_norm=qk_norm)
    eng = ActuationEngine(cfg, 0, seed=0, kv_cache_dtype=kv)
    toks = torch.randint(0, 512, (1, 45), device="cuda:0",
                         generator=torch.Generator("cuda:0").manual_seed(1))
    out = eng.generate(toks, max_new_tokens=60)
    assert eng.stats()["graph_decode"]
    dec = StaticDecoder(eng.model, 1, cfg.max_seq_len)
    assert torch.equal(dec.generate(toks, 60), out)          # eager steps
    eng.sleep()
    eng.wake_up()
    assert torch.equal(eng.generate(toks, max_new_tokens=60), out)
    # logits beside those over a 16-bit cache
    ref = ActuationEngine(cfg, 0, seed=0)
    a = eng.model.forward(toks, eng.new_kv_cache(1, 64), 0)
    b = ref.model.forward(toks, ref.new_kv_cache(1, 64), 0)
    assert (a - b).norm() < 0.1 * b.norm()


def test_tables_of_a_model_longer_than_its_cache():
    from fma_amd.models.llama import LlamaConfig
    from fma_amd.runtime.engine import ActuationEngine
    eng = ActuationEngine(LlamaConfig.tiny_qwen3(), 0, seed=0,
                          kv_cache_dtype="fp8")
    toks = torch.randint(0, 512, (3, 20), device="cuda:0")
    out = eng.model.generate(toks, 30)                        # heads of 16
    assert out.shape == (3, 50)
    with pytest.raises(ValueError, match="tables"):
        eng.model.forward(toks, eng.new_kv_cache(3, 300), 0)


def test_padded_queries_in_front_of_the_last_token(ops):
    c, k, v = filled(ops, 150, B=2, hd=64, cap=200)
    for start, T, counts in ((10, 4, (3, 1)), (0, 150, (150, 40)),
                             (97, 40, (2, 40))):
        q = randn(2, T, 8, 64, seed=T)
        n, s = ints(*counts), ints(start, start)
        outs = [ops.kv8_attention(q, c, 1, start, n),
                ops.kv8_attention(q, c, 1, s, n), ops.kv8_attention(q, c, 1, s)]
        for i, out in enumerate(outs):
            for b, m in enumerate(counts if i < 2 else (T, T)):
                want, bound = oracle.attention(
                    q[b, :m], oracle.held(k[b], "fp8")[:start + m],
                    oracle.held(v[b], "fp8")[:start + m], start, 0.125)
                oracle.check(out[b, :m], want, bound, BF)
                assert not out[b, m:].any()


def test_gradients_of_gains_and_bad_scales_are_refused(ops):
    q = randn(1, 2, 2, 64)
    cos, sin = oracle.tables(10, 64, "cuda")
    w = torch.ones(64, device="cuda", dtype=BF, requires_grad=True)
    c, k, v = filled(ops, 3, hd=64, cap=10)
    for args in ((w, None), (None, w)):
        with pytest.raises(ValueError, match="gradient"):
            ops.fast_qk_norm_rope(q, q, cos, sin, 0, *args)
        with pytest.raises(ValueError, match="gradient"):
            ops.qk_norm_rope_kv8(c, 1, q, q, q, cos, sin, 3, *args)
        with torch.no_grad():
            ops.fast_qk_norm_rope(q, q, cos, sin, 0, *args)
    for scale in (float("nan"), float("inf"), -1e300):
        with pytest.raises(ValueError, match="scale"):
            ops.kv8_attention(q[:, :1], c, 1, 2, scale=scale)


def test_captured_calls_and_lengths_that_the_host_knows(ops):
    """Replays move the cache without the host: what it knew before them does
    not count, and a captured call does not keep what it knew."""
    B, H, cap = 1, 2, 256
    c = ops.KV8Cache(1, B, cap, H, 64, device="cuda")
    k, v = randn(B, cap, H, 64), randn(B, cap, H, 64, seed=1)
    q = randn(B, 1, 4, 64, seed=2)
    at = ints(60)
    kb, vb = torch.zeros_like(k[:, :1]), torch.zeros_like(v[:, :1])

    def check(out, n):
        want, bound = oracle.attention(q[0], oracle.held(k[0, :n], "fp8"),
                                       oracle.held(v[0, :n], "fp8"), n - 1,
                                       0.125)
        oracle.check(out[0], want, bound, BF)

    # attention alone: recorded while the host knows the length, replayed at
    # other ones
    ops.kv8_append(c, 0, k[:, :100], v[:, :100], 0)
    ops.kv8_attention(q, c, 0, at)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.kv8_attention(q, c, 0, at)
        with pytest.raises(ValueError, match="captured"):
            ops.kv8_attention(q, c, 0, 60)
    for n in (100, 61, 200, 96, 130):
        ops.kv8_append(c, 0, k[:, :n], v[:, :n], 0)
        at.fill_(n - 1)
        g.replay()
        check(out, n)
        check(ops.kv8_attention(q, c, 0, at), n)
    # a recorded store: the host knew 40 tokens, replays add 30
    ops.kv8_append(c, 0, k[:, :40], v[:, :40], 0)
    at.fill_(40)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.kv8_append(c, 0, kb, vb, at)
        out = ops.kv8_attention(q, c, 0, at)
    for _ in range(2):
        c.reset()
        ops.kv8_append(c, 0, k[:, :40], v[:, :40], 0)
        for t in range(40, 70):
            at.fill_(t)
            kb.copy_(k[:, t:t + 1])
            vb.copy_(v[:, t:t + 1])
            g.replay()
            check(out, t + 1)
        # by number behind the replays
        ops.kv8_append(c, 0, k[:, 70:75], v[:, 70:75], 70)
        check(ops.kv8_attention(q, c, 0, 74), 75)


def test_read_from_far_behind_the_cache(ops):
    c, k, _ = filled(ops, 40, B=3, hd=64, cap=64)
    junk = [torch.full((1 << 20,), 7.0, device="cuda") for _ in range(4)]
    del junk                                # what outputs would lie in
    start = ints(2 ** 31 - 1, -5, 2 ** 31 - 40)
    rk, rv = ops.kv8_read(c, 1, start, 70, 40)
    assert not rk[0].any() and not rk[2].any()
    assert not rv[0].any() and not rv[2].any()
    assert torch.equal(rk[1, 32:40], k[1, 32:]) and not rk[1, 40:].any()


def test_positions_far_outside_store_and_see_nothing(ops):
    c, k, v = filled(ops, 40, B=3, hd=64, cap=64)
    before = [x.clone() for x in (c.codes, c.scales, c.tail)]
    far = ints(2 ** 31 - 1, -2 ** 31, 65)
    ops.kv8_append(c, 1, k, v, far)
    assert all(torch.equal(a, b)
               for a, b in zip(before, (c.codes, c.scales, c.tail)))
    for T in (1, 40):
        q = randn(3, T, 8, 64, seed=T)
        assert not ops.kv8_attention(q, c, 1, far).any()
        assert not ops.kv8_attention(q, c, 1, far, ints(T, 2 ** 31 - 1,
                                                        -2 ** 31)).any()


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("hd", [160, 192, 256])
@pytest.mark.parametrize("T,n", [(33, 64), (70, 500), (150, 501), (200, 2700)])
def test_attention_wide_heads(ops, fmt, hd, T, n):
    """Many rows at widths over 128: scores that grow from block to block, in
    either half of a block or in both, for some rows; V's scale up and down."""
    k, v = randn(1, n, 2, hd), randn(1, n, 2, hd, seed=1)
    for i in range(0, n, 32):
        v[:, i:i + 32] *= 2.0 ** ((0, 7, -7, 20, 0, -13, 3, -9)[i // 32 % 8])
    q = randn(1, T, 8, hd, seed=2)
    for j, at in enumerate(range(5, n, 23)):  # now in one half, now the other
        k[:, at] = (q[:, T // 2, 1::4] * min(0.3 * (j + 1), 6)).to(BF)
    q[:, :, 2] *= 25
    q[:, 3, 6] = float("nan")
    c = ops.KV8Cache(2, 1, n, 2, hd, fmt=fmt, device="cuda")
    ops.kv8_append(c, 1, k, v, 0)
    out = ops.kv8_attention(q, c, 1, n - T)
    assert torch.isnan(out[0, 3, 6]).all()
    q[:, 3, 6] = 0
    again = attend_and_check(ops, c, q, k, v, n - T)
    out[0, 3, 6] = again[0, 3, 6]
    assert torch.equal(out, again)
    attend_and_check(ops, c, q[:, :, :2], k, v, n - T, scale=-0.2)


# -- small weights beside one that holds the row ------------------------------

@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("B,T,n,H,group", [(2, 1, 773, 2, 8),
                                           (1, 1024, 1024, 32, 1),
                                           (1, 40, 5000, 2, 4)])
def test_attention_first_token_holds_the_rows(ops, fmt, B, T, n, H, group):
    """The first token, whose V is zero, has 2^26 times the weight of each
    other: what the others give has to come out."""
    hd = 64
    scale = hd ** -0.5
    base = randn(1, 1, H, hd, dtype=FP)
    k = randn(B, n, H, hd, dtype=FP, seed=1) * 0.2
    k[:, :1] = base * (18.0 / scale) / base.square().sum(-1, keepdim=True)
    v = 1 + 0.1 * randn(B, n, H, hd, dtype=FP, seed=2)
    v[:, 0] = 0
    k, v = k.to(BF), v.to(BF)
    q = (base.repeat_interleave(group, 2)
         * (1 + 0.05 * randn(B, T, H * group, 1, dtype=FP, seed=3))).to(BF)
    c = ops.KV8Cache(2, B, n, H, hd, fmt=fmt, device="cuda")
    ops.kv8_append(c, 1, k, v, 0)
    out = ops.kv8_attention(q, c, 1, n - T)
    for b in range(B):
        want, bound = oracle.attention_tight(
            q[b], oracle.held(k[b], fmt), oracle.held(v[b], fmt), n - T,
            scale, 2.0 ** (-32 if fmt == "fp8" else -30))
        # the bound says something: the smaller part of what is looked for
        last = (bound[-1] / want[-1].abs()).max()
        assert last < 0.6, last
        oracle.check(out[b], want, bound, BF)


# -- V near the largest value of its type --------------------------------------

SHAPES = [(1, 75, 2, 8, 1), (1, 5000, 2, 8, 1), (150, 300, 2, 8, 1),
          (70, 4000, 2, 12, 1), (200, 3300, 1, 16, 1)]


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("T,n,H,qh,B", SHAPES)
def test_attention_near_the_largest_values(ops, fmt, T, n, H, qh, B):
    """Sums of weights times such values fit fp32 only once divided."""
    c, k, v = filled(ops, n, H=H, B=B, hd=64, fmt=fmt)
    u = torch.rand(v.shape, generator=torch.Generator("cuda").manual_seed(5),
                   device="cuda")
    v = ((0.5 + 0.5 * u) * 3e38).to(BF)
    ops.kv8_append(c, 1, k, v, 0)
    q = randn(B, T, qh, 64, seed=2)
    attend_and_check(ops, c, q, k, v, n - T)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,n,H,qh,B", SHAPES)
def test_attention_saturates(ops, fmt, dtype, T, n, H, qh, B):
    """Codes of the type's largest value stand for a little more; an infinity
    that is still raw counts as that value."""
    most = torch.finfo(dtype).max
    c, k, v = filled(ops, n, H=H, B=B, hd=64, fmt=fmt, dtype=dtype)
    v.fill_(most)
    v[:, :, :, 5] = -most
    v[:, n // 32 * 32:, :, 7] = float("inf")
    ops.kv8_append(c, 1, k, v, 0)
    q = randn(B, T, qh, 64, seed=2, dtype=dtype)
    out = ops.kv8_attention(q, c, 1, n - T).double()
    want = torch.full_like(out, most)
    want[..., 5] = -most
    # weights and codes are off by at most 2^-8 of what they stand for
    assert ((out - want).abs() <= 2.0 ** -7 * most).all()


# -- blocks of V that lie any number of magnitudes apart -----------------------

def one_block_each(n, T, H, qh, hd, span, seed=0):
    """Keys of block j point along axis j, each query row along that of a
    block that it sees, 2^200 above the others; V's blocks lie `span` (log2)
    apart."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")
    blocks = (n + 31) // 32
    side = (200 * 0.6931 * hd ** 0.5) ** 0.5
    k = 0.02 * rand(1, n, H, hd)
    at = torch.arange(n, device="cuda") // 32
    k[:, torch.arange(n, device="cuda"), :, at] += side
    up = torch.rand(blocks, generator=g, device="cuda") \
        * (span[1] - span[0]) + span[0]
    up[0], up[-2] = span[0], span[1]            # the ends among them
    v = (1 + 0.3 * rand(1, n, H, hd)) * torch.exp2(up[at])[:, None, None]
    last = (n - T + torch.arange(T, device="cuda")) // 32
    pick = (torch.rand(T, qh, generator=g, device="cuda")
            * (last[:, None] + 1)).long()
    q = 0.02 * rand(1, T, qh, hd)
    q[0].scatter_add_(2, pick[:, :, None],
                      torch.full((T, qh, 1), side, device="cuda"))
    return q.to(BF), k.to(BF), v.to(BF)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("n,T,H,qh,hd", [(20 * 32 + 7, 1, 1, 16, 64),
                                         (20 * 32 + 7, 40, 2, 16, 64),
                                         (647, 647, 1, 2, 64),
                                         (6 * 32 + 1, 193, 1, 3, 32),
                                         (20 * 32, 3, 2, 8, 256),
                                         (660, 200, 1, 8, 160)])
@pytest.mark.parametrize("span", [(-60, 110), (110, -60), (-20, -2),
                                  (-5, 30)])
def test_attention_over_blocks_of_any_scale(ops, fmt, n, T, H, qh, hd, span):
    """A row gives what its own block gives, whatever blocks that it gives no
    weight, or that come behind it, hold."""
    q, k, v = one_block_each(n, T, H, qh, hd, span)
    c = ops.KV8Cache(2, 1, n, H, hd, fmt=fmt, device="cuda")
    ops.kv8_append(c, 1, k, v, 0)
    out = ops.kv8_attention(q, c, 1, n - T)
    want, bound = oracle.attention_tight(
        q[0], oracle.held(k[0], fmt), oracle.held(v[0], fmt), n - T,
        hd ** -0.5, 2.0 ** -30)
    assert (bound < 0.02 * want.abs().amax(-1, keepdim=True)).all()
    oracle.check(out[0], want, bound, BF)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("T,qh", [(60, 1), (60, 8)])
def test_attention_does_not_see_later_blocks_of_any_scale(ops, fmt, T, qh):
    """Values behind a row, finite and huge, in codes and raw."""
    n, lo = 110, 50
    c, k, v = filled(ops, n, H=1, fmt=fmt)
    q = randn(1, T, qh, 128, seed=2)
    for at in (64, 96):
        vv = v.clone()
        vv[:, at:] *= 2.0 ** 120
        ops.kv8_append(c, 1, k, vv, 0)
        out = ops.kv8_attention(q, c, 1, lo)
        want, bound = oracle.attention_tight(
            q[0], oracle.held(k[0], fmt), oracle.held(vv[0], fmt), lo,
            128 ** -0.5, 2.0 ** -30)
        assert (bound[:at - lo] < 0.05).all()
        oracle.check(out[0], want, bound, BF)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("T,n,H,qh,B", SHAPES[:4])
@pytest.mark.parametrize("qe,ke", [(122, -80), (-118, 100)])
def test_attention_of_queries_near_the_ends_of_the_type(ops, fmt, T, n, H, qh,
                                                        B, qe, ke):
    c, k, v = filled(ops, n, H=H, B=B, hd=64, fmt=fmt)
    k = (randn(B, n, H, 64, dtype=FP, seed=4) * 2.0 ** ke).to(BF)
    ops.kv8_append(c, 1, k, v, 0)
    q = (randn(B, T, qh, 64, dtype=FP, seed=2) * 2.0 ** qe).to(BF)
    attend_and_check(ops, c, q, k, v, n - T, scale=0.125 * 2.0 ** -(qe + ke))


def test_calls_beyond_one_launch_are_refused(ops):
    """2^32 threads; nothing is launched, and the next call is not blamed."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 34 GB for the outputs")
    q = torch.ones(1, 1, 32, 2, dtype=BF, device="cuda") \
        .expand(1, 1 << 27, 32, 2)
    cos, sin = oracle.tables(4, 2, "cuda")
    for _ in range(2):
        with pytest.raises(ValueError, match="beyond one launch"):
            ops.fast_qk_norm_rope(q, q, cos, sin, ints(0))
        assert (torch.ones(1000, device="cuda") * 2).sum().item() == 2000
    torch.cuda.empty_cache()


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("hd", [16, 32])
@pytest.mark.parametrize("B,T,n,H,qh", [(1, 300, 301, 2, 12),
                                        (1, 70, 4000, 2, 12),
                                        (1, 150, 3300, 1, 16),
                                        (1, 1, 5000, 2, 8),
                                        (32, 1, 1500, 2, 64)])
def test_attention_narrow_heads(ops, fmt, hd, B, T, n, H, qh):
    """Many rows and both joins (under 2048 rows and from there on) at a
    width of 32, where one wave of four stages a block."""
    c, k, v = filled(ops, n, H=H, B=B, hd=hd, fmt=fmt)
    q = randn(B, T, qh, hd, seed=2)
    attend_and_check(ops, c, q, k, v, n - T)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("B,T,n", [(4, 1, 75), (4, 1, 700), (2, 1, 5000),
                                   (2, 12, 800)])
def test_attention_of_few_rows_holds_20_bits_of_a_weight(ops, fmt, B, T, n):
    """Two cut-off parts leave less than 2^-10 of 2^-10 of a weight, the
    rounded ones of the raw block less than that."""
    hd, H, qh = 32, 2, 8
    c, k, v = filled(ops, n, H=H, hd=hd, B=B, fmt=fmt, dtype=HF, kscale=0.5)
    q = randn(B, T, qh, hd, seed=2, dtype=HF, scale=0.5)
    out = ops.kv8_attention(q, c, 1, n - T)
    for b in range(B):
        want, bound = oracle.attention_tight(
            q[b], oracle.held(k[b], fmt), oracle.held(v[b], fmt), n - T,
            hd ** -0.5, 2.0 ** -30, 2.0 ** -20)
        oracle.check(out[b], want, bound, HF)
