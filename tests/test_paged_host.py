"""The paged cache and the verification of drafts without a GPU: frequencies, refusals."""
import ctypes
import math

import pytest
import torch

INVALID, UNSUPPORTED = 1, 2


def test_frequencies_match_hf_definitions():
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    from otf_llm.paged import rope_frequencies
    for scaling in ({"rope_type": "linear", "factor": 4.0},
                    {"rope_type": "llama3", "factor": 32.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                     "original_max_position_embeddings": 8192},
                    {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096}):
        cfg = LlamaConfig(hidden_size=512, num_attention_heads=4, head_dim=128, max_position_embeddings=131072,
                          rope_parameters=dict(scaling, rope_theta=500000.0))
        want, factor = ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, "cpu")
        got, mine = rope_frequencies(128, 500000.0, scaling)
        assert got.dtype == torch.float64
        # HF computes in fp32, powers and ramps among it
        assert torch.allclose(got.float(), want, rtol=2e-5, atol=0) and math.isclose(mine, factor, rel_tol=1e-12)
    plain, one = rope_frequencies(128, 500000.0)
    assert one == 1.0 and torch.equal(plain, 500000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128))


def test_frequencies_refuse_what_they_do_not_know():
    from otf_llm.paged import rope_frequencies
    for bad in ({"rope_type": "dynamic", "factor": 2.0}, {"rope_type": "linear"}, {"factor": 2.0},
                {"rope_type": "linear", "factor": -1.0}, {"rope_type": "linear", "factor": 2.0, "mscale": 1.0},
                {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 4.0, "high_freq_factor": 1.0,
                 "original_max_position_embeddings": 8192}):
        with pytest.raises(ValueError):
            rope_frequencies(64, 10000.0, bad)
    for rot, theta in ((63, 1e4), (-2, 1e4), (64, 0.0)):
        with pytest.raises(ValueError):
            rope_frequencies(rot, theta)
    assert rope_frequencies(0)[0].numel() == 0


def test_frequencies_refuse_two_thetas():
    """Dicts that carry rope_theta beside the scaling: it has to be the theta given."""
    from otf_llm.paged import rope_frequencies
    linear = {"rope_type": "linear", "factor": 2.0}
    want = rope_frequencies(64, 500000.0, linear)[0]
    assert torch.equal(rope_frequencies(64, 500000.0, dict(linear, rope_theta=500000))[0], want)
    for kind in (linear, {"rope_type": "default"}):
        with pytest.raises(ValueError, match="rope_theta"):
            rope_frequencies(64, 10000.0, dict(kind, rope_theta=500000.0))


def test_decoders_take_scaled_rotary_tables():
    """rope_table without scaling is HF's default table bit for bit; with it HF's scaled one, within the fp32
    angles that HF computes (an ulp of the angle, and one fp16 rounding)."""
    from transformers import LlamaConfig
    from transformers.models.llama.modeling_llama import LlamaRotaryEmbedding

    from otf_llm.decode_model import ModelConfig, rope_table
    base = dict(layers=1, hidden=256, intermediate=256, heads=2, kv_heads=2, head_dim=128, vocab=10, rope_theta=500000.0,
                max_pos=300)
    scalings = [None, {"rope_type": "linear", "factor": 4.0},
                {"rope_type": "llama3", "factor": 32.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                 "original_max_position_embeddings": 8192},
                {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096}]
    for scaling in scalings:
        hf = LlamaConfig(hidden_size=256, num_attention_heads=2, head_dim=128, max_position_embeddings=131072,
                         rope_parameters=dict(scaling or {"rope_type": "default"}, rope_theta=500000.0))
        x = torch.zeros(1, 300, 256, dtype=torch.float32)
        cos, sin = LlamaRotaryEmbedding(hf)(x, torch.arange(300)[None])
        got = rope_table(ModelConfig(**base, rope_scaling=scaling), "cpu")
        want = torch.stack((cos[0], sin[0]), dim=1)
        if scaling is None:
            assert torch.equal(got, want.half())
        # frequencies of HF within 2e-5 of ours, angles below 300: 6e-3 at most
        assert float((got.float() - want).abs().max()) <= 6.5e-3
    assert torch.equal(rope_table(ModelConfig(**base), "cpu"), rope_table(ModelConfig(**base, rope_scaling=None), "cpu"))


def test_no_cpu_cache():
    from otf_llm.paged import PagedKVCache
    from otf_llm.speculative import verify_drafts
    k = torch.zeros(2, 16, 1, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        PagedKVCache(k, k.clone(), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        verify_drafts(torch.zeros(1, 1, 8), torch.zeros(1, 0, dtype=torch.int64), temperature=0.0)


FAKE = 1 << 20          # never read: every case is refused before anything runs


def cache(**other):
    from otf_llm import _native as N
    c = N.PagedCache()
    given = dict(k_pages=FAKE, v_pages=FAKE, page_stride=16 * 2 * 64, token_stride=128, head_stride=64, n_pages=10,
                 page_size=16, kv_heads=2, head_dim=64, page_table=FAKE, ld_table=4, max_pages=4, lengths=FAKE, batch=3,
                 dtype=0)
    given.update(other)
    for k, v in given.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [(dict(k_pages=None), INVALID), (dict(lengths=None), INVALID), (dict(page_table=None), INVALID),
              (dict(dtype=2), UNSUPPORTED), (dict(head_dim=96), UNSUPPORTED), (dict(batch=0), INVALID),
              (dict(batch=4097), UNSUPPORTED), (dict(page_size=0), INVALID), (dict(n_pages=0), INVALID),
              (dict(kv_heads=0), INVALID), (dict(ld_table=3), INVALID), (dict(k_pages=FAKE + 8), INVALID),
              (dict(token_stride=132), INVALID), (dict(head_stride=56), INVALID), (dict(page_stride=-8), INVALID),
              (dict(max_pages=1 << 30, ld_table=1 << 30), UNSUPPORTED)]


@pytest.mark.parametrize("other,status", BAD_CACHES)
def test_abi_refuses_bad_caches(other, status):
    from otf_llm import _native as N
    L, ref = N.lib(), ctypes.byref(cache(**other))
    good = ctypes.byref(cache())
    assert L.otf_paged_append(ref, None, None, 0, None, 0, 0, FAKE, 128, FAKE, 128, None, None, 3, None) == status
    assert L.otf_paged_attn(ref, FAKE, 256, 4, 1, 1.0, FAKE, 256, None, 0, FAKE, 1 << 40, None) == status
    assert L.otf_paged_evict(ref, good, FAKE, 64, FAKE, 64, 8, 2, FAKE, FAKE, None) == status
    assert L.otf_paged_evict(good, ref, FAKE, 64, FAKE, 64, 8, 2, FAKE, FAKE, None) == status


def test_abi_refuses_bad_arguments():
    from otf_llm import _native as N
    L, c = N.lib(), ctypes.byref(cache())
    rot = N.RotaryArgs()
    rot.turns, rot.rot_dim, rot.factor = FAKE, 64, 1.0

    def append(q=FAKE, ldq=256, qo=FAKE, ldqo=256, heads=4, k=FAKE, ldk=128, v=FAKE, ldv=128, starts=None, n=3, r=rot):
        return L.otf_paged_append(c, ctypes.byref(r) if r is not None else None, q, ldq, qo, ldqo, heads, k, ldk, v, ldv,
                                  starts, None, n, None)
    for bad in (dict(n=4), dict(n=-1), dict(ldq=255), dict(ldq=128), dict(qo=None), dict(heads=0), dict(k=None),
                dict(ldk=64), dict(v=FAKE + 2), dict(ldv=129)):
        assert append(**bad) == INVALID, bad
    assert append(n=0) == 0
    for dims in (63, 66, -2):
        r = N.RotaryArgs()
        r.turns, r.rot_dim = FAKE, dims
        assert append(r=r) == INVALID
    r = N.RotaryArgs()
    r.turns, r.rot_dim = None, 32
    assert append(r=r) == INVALID

    def attn(q=FAKE, ldq=256, heads=4, tokens=1, out=FAKE, ldo=256, w=None, ldw=0, ws=FAKE, n=1 << 40):
        return L.otf_paged_attn(c, q, ldq, heads, tokens, 1.0, out, ldo, w, ldw, ws, n, None)
    for bad in (dict(q=None), dict(out=None), dict(heads=3), dict(heads=0), dict(tokens=0), dict(ldq=248), dict(ldo=250),
                dict(w=FAKE, ldw=63), dict(ws=None), dict(ws=FAKE + 16), dict(n=0)):
        assert attn(**bad) == INVALID, bad
    assert attn(tokens=17) == UNSUPPORTED
    assert L.otf_paged_attn_workspace_bytes(3, 4, 2, 64, 1, 64, 0) > 0
    for bad in ((0, 4, 2, 64, 1, 64, 0), (3, 5, 2, 64, 1, 64, 0), (3, 4, 2, 64, 17, 64, 0), (3, 4, 2, 64, 1, 0, 1)):
        assert L.otf_paged_attn_workspace_bytes(*bad) == -1

    def evict(to=None, w=FAKE, ldw=64, wo=FAKE, ldwo=64, budget=8, recent=2, kept=FAKE, out=FAKE):
        return L.otf_paged_evict(c, ctypes.byref(to) if to is not None else c, w, ldw, wo, ldwo, budget, recent, kept,
                                 out, None)
    for bad in (dict(w=None), dict(wo=None), dict(kept=None), dict(out=None), dict(budget=0), dict(budget=65),
                dict(recent=9), dict(recent=-1), dict(ldw=63), dict(ldwo=32), dict(wo=FAKE + 1024, ldwo=7),
                dict(to=cache(head_dim=128, head_stride=128, token_stride=256)), dict(to=cache(dtype=1)),
                dict(to=cache(page_size=8)), dict(to=cache(batch=2))):
        assert evict(**bad) == INVALID, bad


def test_abi_refuses_bad_verifications():
    from otf_llm import _native as N
    L = N.lib()
    assert L.otf_verify_workspace_bytes(2, 3, 100, 1) == 0
    n = L.otf_verify_workspace_bytes(64, 5, 128256, 1)
    assert n > 0
    for bad in ((0, 3, 100, 0), (2, -1, 100, 0), (2, 33, 100, 0), (2, 3, 0, 0), (65536, 3, 100, 0), (2, 3, (1 << 30) + 1, 0)):
        assert L.otf_verify_workspace_bytes(*bad) == -1

    def verify(t=FAKE, ts=400, ldt=100, d=None, ds=0, ldd=0, tok=FAKE, ldtok=3, u=FAKE, ldu=3, e=FAKE, lde=100, temp=1.0,
               out=FAKE, acc=FAKE, batch=2, drafts=3, vocab=100, ws=None, size=0):
        return L.otf_verify_drafts(t, ts, ldt, d, ds, ldd, tok, ldtok, u, ldu, e, lde, None, temp, None, out, acc, batch,
                                   drafts, vocab, ws, size, None)
    for bad in (dict(t=None), dict(ldt=99), dict(d=FAKE, ldd=99), dict(tok=None), dict(ldtok=2), dict(u=None),
                dict(ldu=2), dict(e=None), dict(lde=99), dict(temp=-1.0), dict(temp=float("nan")),
                dict(temp=float("inf")), dict(temp=1e-30), dict(out=None), dict(acc=None), dict(batch=0),
                dict(drafts=-1), dict(vocab=0)):
        assert verify(**bad) == INVALID, bad
    assert verify(drafts=33, ldtok=33, ldu=33) == UNSUPPORTED
    large = dict(ldt=128256, d=FAKE, ldd=128256, ldtok=5, ldu=5, lde=128256, batch=64, drafts=5, vocab=128256)
    for bad in (dict(ws=None, size=n), dict(ws=FAKE + 8, size=n), dict(ws=FAKE, size=n - 1)):
        assert verify(**large, **bad) == INVALID, bad


def test_attention_workspace_does_not_wrap():
    """The scores' scratch of the largest tables passes 64 bits as a product: it is refused, or so large that
    no small workspace is taken for it."""
    from otf_llm import _native as N
    L = N.lib()
    for batch, heads, kv, tokens, most in ((4096, 65535, 1, 16, 1 << 30), (4096, 64512, 1024, 16, 1 << 30),
                                           (4095, 65535, 1, 16, 1 << 29), (4096, 32768, 512, 16, 1 << 30)):
        n = L.otf_paged_attn_workspace_bytes(batch, heads, kv, 64, tokens, most, 1)
        assert n == -1 or n >= heads // kv * tokens * most * 4
        c = cache(batch=batch, kv_heads=kv, token_stride=kv * 64, page_stride=16 * kv * 64, max_pages=most // 16,
                  ld_table=most // 16)
        for size in (0, 1 << 20, 1 << 30):
            # (device memory of this size is never read: no GPU, or refused before)
            assert L.otf_paged_attn(ctypes.byref(c), FAKE, heads * 64, heads, tokens, 1.0, FAKE, heads * 64, FAKE, most, FAKE,
                                    size, None) in (INVALID, UNSUPPORTED)
    for bad in ((4097, 4, 2, 64, 1, 64, 0), (1, 65536, 1, 64, 1, 64, 0), (1, 1025, 1025, 64, 1, 64, 0),
                (1, 4, 2, 96, 1, 64, 0), (1, 4, 2, 64, 1, (1 << 30) + 1, 0), (1 << 40, 1 << 40, 1, 64, 1, 1 << 40, 1)):
        assert L.otf_paged_attn_workspace_bytes(*bad) == -1, bad


def test_abi_refuses_scales_that_are_not_finite():
    """Nor finite times log2(e), which the scores' exponents are taken with."""
    from otf_llm import _native as N
    L, c = N.lib(), ctypes.byref(cache())
    for scale in (float("inf"), -float("inf"), float("nan"), 3e38, -2.4e38):
        assert L.otf_paged_attn(c, FAKE, 256, 4, 1, scale, FAKE, 256, None, 0, FAKE, 1 << 40, None) == INVALID


def test_attention_workspace_is_bounded():
    """Scratch for the scores of tables with much room: 2 GiB at most, or one KV head's; small calls as before."""
    from otf_llm import _native as N
    f = N.lib().otf_paged_attn_workspace_bytes
    for batch, heads, kv, tokens, most in ((64, 64, 8, 16, 131072), (64, 64, 8, 1, 131072), (4096, 8, 8, 5, 8192),
                                           (1, 128, 8, 16, 1 << 20), (3, 128, 4, 16, 1 << 20)):
        one = heads // kv * tokens * most * 4
        plain = f(batch, heads, kv, 128, tokens, most, 0)
        assert plain <= 16 << 20
        assert plain + one <= f(batch, heads, kv, 128, tokens, most, 1) <= plain + max(one, 2 << 30) + (8 << 20)
    n = f(16, 32, 8, 128, 5, 4020, 1) - f(16, 32, 8, 128, 5, 4020, 0)
    assert 16 * 8 * 20 * 4020 * 4 <= n <= 16 * 8 * 20 * 4020 * 4 + 16 * 8 * 20 * 4 + 512


def test_abi_append_with_weights_refuses():
    from otf_llm import _native as N
    L, c = N.lib(), ctypes.byref(cache())

    def append(w=FAKE, ldw=64, n=3, k=FAKE):
        return L.otf_paged_append_weights(c, None, None, 0, None, 0, 0, k, 128, FAKE, 128, None, None, n, w, ldw, None)
    assert append(n=0) == 0
    assert append(ldw=63) == INVALID and append(n=4) == INVALID and append(k=None) == INVALID


def overlaps(x, ldx, colx, y, ldy, coly, rows):
    """Element by element."""
    return bool({x + i * ldx + c for i in range(rows) for c in range(colx)} &
                {y + i * ldy + c for i in range(rows) for c in range(coly)})


def test_abi_refuses_outputs_over_inputs():
    """Queries and outputs in one buffer that share an element, as counted one by one (those that share none
    are called on a GPU)."""
    import random

    from otf_llm import _native as N
    L, c = N.lib(), cache(batch=5)
    base, far, rng, seen = 1 << 40, 1 << 41, random.Random(3), 0
    for _ in range(600):
        ldq = ldo = 8 * rng.randint(32, 80)
        if rng.random() < 0.4:
            ldo = 8 * rng.randint(32, 80)
        delta = 8 * rng.randint(-5 * 60, 5 * 60)
        if overlaps(0, ldq, 256, delta, ldo, 256, 5):
            seen += 1
            assert L.otf_paged_attn(ctypes.byref(c), base, ldq, 4, 1, 1.0, base + 2 * delta, ldo, None, 0, FAKE, 1 << 40,
                                    None) == INVALID, (ldq, ldo, delta)
            if delta or ldq != ldo:                         # append's q_out may be q
                assert L.otf_paged_append(ctypes.byref(c), None, base, ldq, base + 2 * delta, ldo, 4, far, 128, far, 128, None,
                                          None, 5, None) == INVALID, (ldq, ldo, delta)
        if overlaps(0, ldq, 128, delta, ldo, 256, 5):       # keys and values have 128 columns
            for k, v in ((base, far), (far, base)):
                assert L.otf_paged_append(ctypes.byref(c), None, far, 256, base + 2 * delta, ldo, 4, k, ldq, v, ldq, None, None, 5,
                                          None) == INVALID, (ldq, ldo, delta)
    assert seen > 200


def test_abi_refuses_evictions_over_their_inputs():
    from otf_llm import _native as N
    L, c = N.lib(), cache()
    to = cache(page_table=FAKE + 4096)
    w, far = 1 << 40, 1 << 41                               # weights: 3 x 2 x 64 numbers

    def evict(t, wo, ldwo=64, out=far):
        return L.otf_paged_evict(ctypes.byref(c), ctypes.byref(t), w, 64, wo, ldwo, 8, 2, far + (1 << 20), out, None)
    for wo in (w + 4, w - 4, w + 4 * 3 * 2 * 64 - 4, w - 4 * 3 * 2 * 64 + 4):
        assert evict(to, wo) == INVALID
    assert evict(to, w - 4 * 3 * 2 * 40 + 4, 40) == INVALID
    for out in (FAKE + 4, FAKE - 8, FAKE):
        assert evict(to, far + 4096, out=out) == INVALID
    for out in (FAKE + 4, FAKE - 8):
        assert evict(c, w, out=out) == INVALID


# lengths, query heads, KV heads, head size: few tokens, where a probability's rounding shows, and some hundred
# nearly equal ones, where a lost one does
SHARP = [(2, 8, 2, 64), (5, 16, 4, 128), (17, 8, 1, 64), (300, 8, 2, 64), (611, 16, 2, 128)]


def sharp_inputs(n, heads, kv, dim, dtype):
    g = torch.Generator().manual_seed(n)
    q = (0.3 * torch.randn(heads, dim, generator=g)).to(dtype)
    k, v = (torch.randn(n, kv, dim, generator=g).to(dtype) for _ in range(2))
    return q, k, v


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,heads,kv,dim", SHARP)
def test_attention_tolerance_tells_mistakes(n, heads, kv, dim, dtype):
    """The bound that the attention is held to admits probabilities of two 16-bit numbers, and not a rest left
    out or exchanged (where few tokens share the mass) nor a token lost."""
    import paged_oracle as ref
    q, k, v = sharp_inputs(n, heads, kv, dim, dtype)
    k, v = k.double(), v.double()
    y, p, mass, size = ref.attend(q, k, v, dim ** -0.5)
    tol = ref.attend_tolerance_two(y, mass, size, dim, dtype, n, float(v.abs().max()))

    def off(**mistake):
        return float(((ref.attend_as_products_see(q, k, v, dim ** -0.5, dtype, **mistake) - y).abs() / tol).max())
    assert off() <= 1
    for lost in (0, n // 2, n - 1):
        assert off(lost=lost) > 2
    if n <= 17:
        assert off(rest=False) > 2 and off(turned=True) > 2
