"""The 8-bit cache and norm + rotation on the CPU: formulas, bookkeeping and
refusals."""

import pytest
import torch

from fma_amd.ops.decode_ops import fast_qk_norm_rope
from fma_amd.ops.kv8 import (KV8Cache, kv8_append, kv8_attention, kv8_read,
                             qk_norm_rope_kv8)
from tests import kv8_oracle as oracle


def make(fmt="fp8", dtype=torch.bfloat16, B=1, S=100, H=2, hd=16, layers=1):
    return KV8Cache(layers, B, S, H, hd, fmt=fmt, dtype=dtype)


def value(x, dtype):
    """A held value as kv8_read gives it: the product of code and scale is
    exact in 64 bits, so this is its fp32 rounding and then the type's."""
    return x.float().to(dtype)


def kv(T, B=1, H=2, hd=16, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(B, T, H, hd, generator=g) * 3
    v = torch.randn(B, T, H, hd, generator=g)
    return k.to(dtype), v.to(dtype)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_read_gives_what_the_definition_says(fmt, dtype):
    c = make(fmt, dtype, hd=20)
    k, v = kv(75, hd=20, dtype=dtype)
    kv8_append(c, 0, k, v, 0)
    rk, rv = kv8_read(c, 0, 0, 80, 75)
    assert torch.equal(rk[0, :75], value(oracle.held(k[0], fmt), dtype))
    assert torch.equal(rv[0, :75], value(oracle.held(v[0], fmt), dtype))
    assert not rk[0, 75:].any() and not rv[0, 75:].any()


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_result_does_not_depend_on_how_tokens_arrive(fmt):
    k, v = kv(97)
    whole, parts = make(fmt), make(fmt)
    kv8_append(whole, 0, k, v, 0)
    at = 0
    for n in (1, 30, 1, 5, 40, 3, 17):
        kv8_append(parts, 0, k[:, at:at + n], v[:, at:at + n], at)
        at += n
    for a, b in zip(kv8_read(whole, 0, 0, 97, 97),
                    kv8_read(parts, 0, 0, 97, 97)):
        assert torch.equal(a, b)


def test_not_finite_values():
    c = make()
    k, v = kv(40)
    k[0, 3, 0, 1], k[0, 4, 1, 2] = float("nan"), float("inf")
    v[0, 5, 0, 0] = float("-inf")
    kv8_append(c, 0, k, v, 0)
    rk, rv = kv8_read(c, 0, 0, 32, 40)
    assert rk[0, 3, 0, 1] == 0
    assert torch.equal(rk[0], value(oracle.held(k[0, :32], "fp8"), k.dtype))
    assert torch.equal(rv[0], value(oracle.held(v[0, :32], "fp8"), v.dtype))


def test_zero_block_and_tiny_values():
    for fmt in ("fp8", "int8"):
        c = make(fmt)
        k = torch.zeros(1, 32, 2, 16, dtype=torch.bfloat16)
        v = torch.full_like(k, 2.0 ** -110)
        kv8_append(c, 0, k, v, 0)
        rk, rv = kv8_read(c, 0, 0, 32, 32)
        assert not rk.any()
        assert torch.equal(rv[0], value(oracle.held(v[0], fmt), v.dtype))


def test_going_back_after_a_rejected_draft():
    k, v = kv(80)
    c = make()
    kv8_append(c, 0, k[:, :62], v[:, :62], 0)
    junk_k, junk_v = kv(5, seed=9)
    kv8_append(c, 0, junk_k, junk_v, 62)     # completes a block, with junk
    kv8_append(c, 0, k[:, 62:80], v[:, 62:80], 62)
    ref = make()
    kv8_append(ref, 0, k, v, 0)
    for a, b in zip(kv8_read(c, 0, 0, 80, 80), kv8_read(ref, 0, 0, 80, 80)):
        assert torch.equal(a, b)


def test_later_block_in_the_slot_of_the_first():
    """One call that reads a block's earlier tokens and ends in a block that
    is held in the same slot."""
    for end in (70, 96, 97, 130):
        k, v = kv(end)
        c, ref = make(S=200), make(S=200)
        kv8_append(c, 0, k[:, :5], v[:, :5], 0)
        kv8_append(c, 0, k[:, 5:], v[:, 5:], 5)
        kv8_append(ref, 0, k, v, 0)
        for a, b in zip(kv8_read(c, 0, 0, end, end),
                        kv8_read(ref, 0, 0, end, end)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("T", [1, 3, 40])
def test_attention_matches_the_oracle(fmt, T):
    k, v = kv(90)
    c = make(fmt)
    kv8_append(c, 0, k, v, 0)
    q = torch.randn(1, T, 6, 16, generator=torch.Generator().manual_seed(3)) \
        .bfloat16()
    out = kv8_attention(q, c, 0, 90 - T)
    want, bound = oracle.attention(q[0], oracle.held(k[0], fmt),
                                   oracle.held(v[0], fmt), 90 - T, 0.25)
    oracle.check(out[0], want, bound, q.dtype)


def test_queries_in_front_of_the_last_token():
    k, v = kv(150)
    c = make(S=200)
    kv8_append(c, 0, k, v, 0)
    for start, T in ((49, 1), (40, 30), (0, 3), (127, 2), (95, 1)):
        q = torch.randn(1, T, 4, 16).bfloat16()
        out = kv8_attention(q, c, 0, start)
        n = start + T
        want, bound = oracle.attention(
            q[0], oracle.held(k[0], "fp8")[:n], oracle.held(v[0], "fp8")[:n],
            start, 0.25)
        oracle.check(out[0], want, bound, q.dtype)


def test_ragged_batch():
    k, v = kv(50, B=3)
    c = make(B=3)
    start = torch.tensor([0, 0, 0], dtype=torch.int32)
    counts = torch.tensor([50, 0, 33], dtype=torch.int32)
    kv8_append(c, 0, k, v, start, counts)
    q = torch.randn(3, 50, 2, 16).bfloat16()
    out = kv8_attention(q, c, 0, start, counts)
    assert not out[1].any() and not out[2, 33:].any()
    for b, n in ((0, 50), (2, 33)):
        want, bound = oracle.attention(
            q[b, :n], oracle.held(k[b, :n], "fp8"),
            oracle.held(v[b, :n], "fp8"), 0, 0.25)
        oracle.check(out[b, :n], want, bound, q.dtype)


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("rot,norm", [(16, True), (10, True), (6, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16,
                                   torch.float32])
def test_norm_rope_matches_the_oracle(interleaved, rot, norm, dtype):
    g = torch.Generator().manual_seed(1)
    q = torch.randn(2, 5, 4, 16, generator=g).to(dtype)
    k = torch.randn(2, 5, 2, 16, generator=g).to(dtype)
    cos, sin = oracle.tables(50, rot, factor=1.2)
    w = [torch.rand(16, generator=g).to(dtype) if norm else None
         for _ in range(2)]
    pos = torch.randint(0, 50, (2, 5), generator=g)
    got = fast_qk_norm_rope(q, k, cos, sin, pos, *w, interleaved=interleaved)
    for x, y, g_ in zip((q, k), got, w):
        want, bound = oracle.norm_rope(x, g_, cos, sin, pos, 1e-6,
                                       interleaved)
        oracle.check(y, want, bound, dtype)


def test_norm_rope_position_forms_and_outside():
    q, k = torch.randn(2, 3, 2, 8), torch.randn(2, 3, 1, 8)
    cos, sin = oracle.tables(10, 8)
    a = fast_qk_norm_rope(q, k, cos, sin, 4)
    b = fast_qk_norm_rope(q, k, cos, sin, torch.tensor([4, 4]))
    c = fast_qk_norm_rope(q, k, cos, sin,
                          torch.tensor([[4, 5, 6]] * 2, dtype=torch.int32))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], c[1])
    d = fast_qk_norm_rope(q, k, cos, sin, torch.tensor([8, -1]))
    assert torch.isnan(d[0][0, 2]).all() and torch.isnan(d[1][1, 0]).all()
    assert torch.isfinite(d[0][0, :2]).all()


def test_one_call_is_the_two_calls():
    q = torch.randn(1, 40, 4, 16).bfloat16()
    k, v = kv(40)
    cos, sin = oracle.tables(100, 16)
    w = torch.rand(16).bfloat16()
    a, b = make(), make()
    qa = qk_norm_rope_kv8(a, 0, q, k, v, cos, sin, 0, w, w)
    qb, kb = fast_qk_norm_rope(q, k, cos, sin, 0, w, w)
    kv8_append(b, 0, kb, v, 0)
    assert torch.equal(qa, qb)
    for x, y in zip(kv8_read(a, 0, 0, 40, 40), kv8_read(b, 0, 0, 40, 40)):
        assert torch.equal(x, y)


def test_refusals_of_the_cache():
    for bad in (dict(fmt="int4"), dict(dtype=torch.float32), dict(hd=257),
                dict(hd=0), dict(S=0), dict(B=0)):
        with pytest.raises(ValueError):
            make(**bad)
    c = make()
    k, v = kv(10)
    for args in ((1, k, v, 0), (-1, k, v, 0), (0, k[..., :8], v, 0),
                 (0, k.float(), v, 0), (0, k[:, :, :1], v, 0),
                 (0, k, v[:, :5], 0), (0, k, v, -1), (0, k, v, 91),
                 (0, k, v, 5), (0, k[0], v, 0),
                 (0, k, v, torch.tensor([0])),
                 (0, k, v, torch.tensor([0, 0], dtype=torch.int32)),
                 (0, k, v, 0, torch.tensor([3]))):
        with pytest.raises(ValueError):
            kv8_append(c, *args)
    with pytest.raises(ValueError):
        kv8_append(c, 0, k.float().requires_grad_().bfloat16(), v, 0)
    kv8_append(c, 0, k, v, 0)
    q = torch.randn(1, 1, 2, 16).bfloat16()
    for args in ((q, c, 0, 10), (q, c, 0, 100), (q, c, 3, 9),
                 (q.float(), c, 0, 9), (q[:, :, :1], c, 0, 9)):
        with pytest.raises(ValueError):
            kv8_attention(*args)
    for args in ((0, 0, -1, 10), (0, 101, 1, 10), (0, 0, 1, 101),
                 (0, 0, 1, 9)):
        with pytest.raises(ValueError):
            kv8_read(c, *args)
    c.free()
    with pytest.raises(ValueError):
        kv8_append(c, 0, k, v, 0)


def test_refuses_to_build_on_values_it_no_longer_holds():
    c = make(S=300)
    k, v = kv(200)
    kv8_append(c, 0, k, v, 0)                 # blocks 5 and 6 are raw
    one = kv(1)
    for start in (159, 100, 33):
        with pytest.raises(ValueError, match="raw values"):
            kv8_append(c, 0, *one, start)
    with pytest.raises(ValueError, match="hole"):
        kv8_append(c, 0, *one, 201)
    kv8_append(c, 0, *one, 161)               # one block back
    with pytest.raises(ValueError, match="holds 162"):
        kv8_attention(torch.zeros(1, 1, 2, 16).bfloat16(), c, 0, 162)
    with pytest.raises(ValueError, match="raw values"):
        kv8_append(c, 0, *one, 159)
    kv8_append(c, 0, *one, 128)               # a block's first token
    kv8_append(c, 0, *one, 129)
    with pytest.raises(ValueError, match="raw values"):
        kv8_append(c, 0, *one, 127)
    c.reset()
    kv8_append(c, 0, *one, 0)


def test_refusals_of_norm_rope():
    q, k = torch.randn(1, 2, 2, 8), torch.randn(1, 2, 1, 8)
    cos, sin = oracle.tables(10, 8)
    w = torch.ones(8)
    for args in ((q[0], k[0], cos, sin, 0), (q, k[:, :1], cos, sin, 0),
                 (q, k.half(), cos, sin, 0), (q, k, cos, sin[:5], 0),
                 (q, k, cos.half(), sin.half(), 0),
                 (q, k, *oracle.tables(10, 10), 0), (q, k, cos, sin, 9),
                 (q, k, cos, sin, -1), (q, k, cos, sin, torch.zeros(2).long()),
                 (q, k, cos, sin, torch.zeros(1)),
                 (q, k, cos, sin, 0, w[:4]), (q, k, cos, sin, 0, w.half()),
                 (q.requires_grad_(), k, cos, sin, 0)):
        with pytest.raises(ValueError):
            fast_qk_norm_rope(*args)
    c = make(hd=8)
    kk, v = kv(2, hd=8)
    with pytest.raises(ValueError, match="tables"):
        qk_norm_rope_kv8(c, 0, torch.zeros(1, 2, 2, 8).bfloat16(), kk, v,
                         cos, sin, 0)


# -- the framework's own paths over it -------------------------------------------

def _generate(cfg, kv, prompt, n=8, batch=1):
    from fma_amd.runtime.engine import ActuationEngine
    eng = ActuationEngine(cfg, seed=0, kv_cache_dtype=kv)
    return eng, eng.generate(prompt.repeat(batch, 1), max_new_tokens=n)


@pytest.mark.parametrize("preset", ["tiny", "tiny_qwen3", "tiny_gemma",
                                    "tiny_moe"])
@pytest.mark.parametrize("kv", ["fp8", "int8"])
def test_families_generate_over_an_8bit_cache(preset, kv):
    """Logits stay near those over a 16-bit cache; prompts of one call and of
    several, and single tokens, agree with each other."""
    from fma_amd.models.llama import LlamaConfig
    from fma_amd.runtime.engine import ActuationEngine
    cfg = getattr(LlamaConfig, preset)()
    a, b = (ActuationEngine(cfg, seed=0, kv_cache_dtype=x)
            for x in ("auto", kv))
    assert b.stats()["kv_cache_dtype"] == kv
    toks = torch.randint(0, cfg.vocab_size, (2, 70),
                         generator=torch.Generator().manual_seed(1))
    ca, cb = a.new_kv_cache(2, 80), b.new_kv_cache(2, 80)
    assert isinstance(cb, KV8Cache) and cb.fmt == kv
    la = a.model.forward(toks, ca, 0)
    lb = b.model.forward(toks, cb, 0)
    # a key or value moves by at most 2^-4 of its size, two layers deep;
    # a wrong token, position or head moves the logits by their own size
    assert (la - lb).norm() < 0.1 * la.norm()
    # rows over whole blocks do not depend on the split of the prompt
    cc = b.new_kv_cache(2, 80)
    b.model.forward(toks[:, :64], cc, 0)
    lc = b.model.forward(toks[:, 64:], cc, 64)
    assert (lc - lb[:, 64:]).norm() < 2e-2 * lb[:, 64:].norm()
    out = b.generate(toks, max_new_tokens=5)
    assert out.shape == (2, 75)


def test_static_decoder_over_an_8bit_cache():
    from fma_amd.models.decode_graph import StaticDecoder
    from fma_amd.models.llama import LlamaConfig
    for cfg in (LlamaConfig.tiny(), LlamaConfig.tiny_qwen3()):
        eng, want = _generate(cfg, "fp8", torch.arange(1, 31)[None], 40)
        assert StaticDecoder.supported(cfg, "fp8")
        dec = StaticDecoder(eng.model, 1, 128)
        for _ in range(2):
            assert torch.equal(dec.generate(torch.arange(1, 31)[None], 40),
                               want)


def test_option_reaches_the_engine():
    from fma_amd.models.llama import LlamaConfig
    from fma_amd.runtime.engine import ActuationEngine
    from fma_amd.runtime.server import ServingRuntime, parse_options
    assert parse_options("--model tiny").kv_cache_dtype == "auto"
    for given, want in (("fp8", "fp8"), ("fp8_e4m3", "fp8"),
                        ("int8", "int8"), ("fp8_e5m2", "auto")):
        args = parse_options(f"--model tiny --kv-cache-dtype {given}")
        assert args.kv_cache_dtype == want
    rt = ServingRuntime(parse_options("--model tiny --kv-cache-dtype fp8"))
    try:
        assert rt.rt.stats()["kv_cache_dtype"] == "fp8"
        assert len(rt.rt.generate_text("hello", 3)) >= 0
    finally:
        rt.close()
    with pytest.raises(ValueError):
        ActuationEngine(LlamaConfig.tiny(), kv_cache_dtype="int4")
    cfg = LlamaConfig.tiny()
    cfg.dtype = torch.float32
    with pytest.raises(ValueError):
        ActuationEngine(cfg, kv_cache_dtype="fp8")


def test_padded_queries_in_front_of_the_last_token():
    """Counts and a tensor of starts say nothing of what is coded where the
    cache knows its length."""
    k, v = kv(150, B=2)
    c = make(S=200, B=2)
    kv8_append(c, 0, k, v, 0)
    for start, T, counts in ((10, 4, (3, 1)), (0, 150, (150, 40)),
                             (97, 40, (2, 40))):
        q = torch.randn(2, T, 4, 16).bfloat16()
        n = torch.tensor(counts, dtype=torch.int32)
        s = torch.full((2,), start, dtype=torch.int32)
        outs = [kv8_attention(q, c, 0, start, n),
                kv8_attention(q, c, 0, s, n)]
        outs.append(kv8_attention(q, c, 0, s))
        for i, out in enumerate(outs):
            for b, m in enumerate(counts if i < 2 else (T, T)):
                want, bound = oracle.attention(
                    q[b, :m], oracle.held(k[b], "fp8")[:start + m],
                    oracle.held(v[b], "fp8")[:start + m], start, 0.25)
                oracle.check(out[b, :m], want, bound, q.dtype)
                assert not out[b, m:].any()


def test_gradients_of_gains_and_bad_scales_are_refused():
    q, k = torch.randn(1, 2, 2, 8), torch.randn(1, 2, 1, 8)
    cos, sin = oracle.tables(10, 8)
    w = torch.ones(8, requires_grad=True)
    for args in ((w, None), (None, w)):
        with pytest.raises(ValueError, match="gradient"):
            fast_qk_norm_rope(q, k, cos, sin, 0, *args)
        with torch.no_grad():
            fast_qk_norm_rope(q, k, cos, sin, 0, *args)
    c = make()
    kk, v = kv(3)
    kv8_append(c, 0, kk, v, 0)
    one = torch.zeros(1, 1, 2, 16).bfloat16()
    for scale in (float("nan"), float("inf"), -1e300):
        with pytest.raises(ValueError, match="scale"):
            kv8_attention(one, c, 0, 2, scale=scale)


def test_option_does_not_keep_a_model_from_being_served(monkeypatch, capsys):
    """Heads that no 8-bit cache holds, and an option without a value."""
    from fma_amd.models.llama import LlamaConfig
    from fma_amd.runtime.server import ServingRuntime, parse_options
    args = parse_options("--model tiny --kv-cache-dtype --seed 3")
    assert (args.kv_cache_dtype, args.seed) == ("auto", 3)

    def wide(name):
        cfg = LlamaConfig.tiny()
        cfg.head_dim_override = 288
        return cfg
    monkeypatch.setattr(LlamaConfig, "by_name", staticmethod(wide))
    rt = ServingRuntime(parse_options("--model tiny --kv-cache-dtype int8"))
    try:
        assert rt.rt.stats()["kv_cache_dtype"] == "auto"
        assert "using auto" in capsys.readouterr().out
        assert len(rt.rt.generate_text("hello", 3)) >= 0
    finally:
        rt.close()


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_saturates(fmt, dtype):
    """Codes of the type's largest value stand for a little more; an infinity
    that is still raw counts as that value."""
    most = torch.finfo(dtype).max
    for T, n in ((1, 75), (20, 40), (3, 3)):
        k, v = kv(n, dtype=dtype)
        v.fill_(most)
        v[..., 5] = -most
        v[:, n // 32 * 32:, :, 7] = float("inf")
        c = make(fmt, dtype)
        kv8_append(c, 0, k, v, 0)
        out = kv8_attention(torch.randn(1, T, 4, 16).to(dtype), c, 0,
                            n - T).double()
        want = torch.full_like(out, most)
        want[..., 5] = -most
        assert ((out - want).abs() <= 2.0 ** -7 * most).all()
