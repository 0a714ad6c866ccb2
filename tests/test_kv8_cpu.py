"""The 8-bit cache without a GPU: what the entry points refuse, and the restatement's own format."""

import pytest
import torch

import plain_kv8 as P
from redline_b200.ops import kernels
from redline_b200.ops.kernels import KernelError

HEADS, KV, DIM, PAGE, PAGES = 4, 2, 64, 16, 5


def cache(**change):
    t = dict(kcache=torch.zeros(PAGES, KV, PAGE, DIM, dtype=torch.uint8).view(P.E4M3),
             vcache=torch.zeros(PAGES, KV, PAGE, DIM, dtype=torch.uint8).view(P.E4M3),
             kscale=torch.zeros(PAGES, KV, dtype=torch.uint8).view(P.E8M0),
             vscale=torch.zeros(PAGES, KV, dtype=torch.uint8).view(P.E8M0))
    t.update(change)
    return t


def ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def write(n=3, **change):
    a = dict(qkv=torch.zeros(n, (HEADS + 2 * KV) * DIM), positions=ints(n), slots=ints(n), cos=torch.zeros(8, DIM // 2),
             sin=torch.zeros(8, DIM // 2), **cache(), q_out=torch.zeros(n, HEADS * DIM), num_heads=HEADS, num_kv_heads=KV,
             head_dim=DIM, page_size=PAGE, status=ints(1))
    a.update(change)
    kernels.kv8_write(**a)


def prefill(n=3, **change):
    a = dict(q=torch.zeros(n, HEADS * DIM), q_stride=HEADS * DIM, **cache(), block_table=ints(2, 4), tile_seq=ints(1), tile_tok=ints(1),
             tile_rows=ints(1), positions=ints(n), out=torch.zeros(n, HEADS * DIM), tiles=1, num_heads=HEADS, num_kv_heads=KV,
             head_dim=DIM, page_size=PAGE, window=0, scale=1.0)
    a.update(change)
    kernels.kv8_attn_prefill(**a)


ODD = [
    (dict(kcache=torch.zeros(PAGES, KV, PAGE, DIM)), "float8_e4m3fn"),
    (dict(kscale=torch.zeros(PAGES, KV)), "float8_e8m0fnu"),
    (dict(page_size=48), "pages of 16, 32 or 64"),
    (dict(page_size=32), "caches"),
    (dict(num_kv_heads=3), "no multiple"),
    (dict(num_kv_heads=0), "no multiple"),
    (dict(num_kv_heads=4), "caches"),
    (dict(vcache=torch.zeros(PAGES + 1, KV, PAGE, DIM, dtype=torch.uint8).view(P.E4M3)), "caches"),
    (dict(vscale=torch.zeros(PAGES, KV + 1, dtype=torch.uint8).view(P.E8M0)), "scales"),
    (dict(kcache=torch.zeros(PAGES, PAGE, KV, DIM, dtype=torch.uint8).transpose(1, 2).view(P.E4M3)), "contiguous"),
    (dict(kcache=torch.zeros(PAGES * KV * PAGE * DIM + 8, dtype=torch.uint8)[8:].view(PAGES, KV, PAGE, DIM).view(P.E4M3)), "16-byte"),
    (dict(), "no CPU fallback"),
]


@pytest.mark.parametrize("change,match", ODD)
def test_caches_that_are_refused(change, match):
    for call in (write, prefill):
        with pytest.raises(KernelError, match=match):
            call(**change)


def test_rows_that_are_refused(monkeypatch):
    """What comes behind the look at the cache (stood in for: there is no device here)."""
    monkeypatch.setattr(kernels, "_kv8_check", lambda *a: None)
    wide = (HEADS + 2 * KV) * DIM
    bad = [
        (write, dict(qkv=torch.zeros(3, wide - 1)), "rows of"),
        (write, dict(qkv=torch.zeros(3, wide + 2)[:, :wide]), "16-byte"),
        (write, dict(qkv=torch.zeros(3, wide + 4)[:, 1:1 + wide]), "16-byte"),
        (write, dict(qkv=torch.zeros(wide, 3).t()), "contiguous"),
        (write, dict(positions=torch.zeros(3, dtype=torch.int64)), "positions must be"),
        (write, dict(positions=ints(2)), "3 tokens"),
        (write, dict(tokens=4), "4 tokens"),
        (write, dict(tokens=-1), "tokens"),
        (write, dict(slots=ints(2)), "2 slots"),
        (write, dict(slots=torch.zeros(3, dtype=torch.int64)), "slots must be"),
        (write, dict(cos=None), "come together"),
        (write, dict(cos=torch.zeros(8, DIM)), "cos / sin"),
        (write, dict(sin=torch.zeros(7, DIM // 2)), "cos / sin"),
        (write, dict(q_out=torch.zeros(2, HEADS * DIM)), "q_out"),
        (write, dict(q_out=torch.zeros(3, HEADS * DIM, dtype=torch.bfloat16)), "q_out"),
        (prefill, dict(q_stride=HEADS * DIM + 8), "apart"),
        (prefill, dict(out=torch.zeros(3, HEADS * DIM, dtype=torch.bfloat16)), "out must be"),
        (prefill, dict(tiles=2), "for 2 tiles"),
        (prefill, dict(window=-1), "window"),
        (prefill, dict(impl=2), "impl 2"),
        (prefill, dict(scale=0.0), "scale must be positive"),
        (prefill, dict(scale=-1.0), "scale must be positive"),
        (prefill, dict(scale=float("nan")), "scale must be positive"),
        (prefill, dict(block_table=ints(8)), "block_table"),
        (prefill, dict(block_table=torch.zeros(2, 4, dtype=torch.int64)), "block_table"),
    ]
    for call, change, match in bad:
        with pytest.raises(KernelError, match=match):
            call(**change)


def test_types_and_sizes_that_are_refused(monkeypatch):
    monkeypatch.setattr(kernels, "_kv8_check", lambda *a: None)
    with pytest.raises(KernelError, match="head sizes"):
        write(qkv=torch.zeros(3, (HEADS + 2 * KV) * 72), head_dim=72, cos=None, sin=None, q_out=None)
    monkeypatch.setattr(kernels, "_kv8", lambda head_dim: None)
    monkeypatch.setattr(kernels, "_fn", lambda lib, name, types: None)
    monkeypatch.setattr(kernels, "_on", lambda t: kernels._here)
    with pytest.raises(KernelError, match="not supported"):
        write(qkv=torch.zeros(3, (HEADS + 2 * KV) * DIM, dtype=torch.float16), q_out=None)


def test_the_formats_borders():
    assert P.code_of(0.0) == 1 and P.code_of(448.0) == 127 and P.code_of(448.0001) == 128 and P.code_of(1.0) == 119
    assert P.code_of(1.75) == 119 and P.code_of(3.4e38) == 246 and P.code_of(1e-44) == 1
    g = torch.Generator().manual_seed(0)
    for size in (1e-30, 1.0, 3e20):
        x = torch.randn(16, 2, 64, generator=g) * size
        cache, scale = torch.zeros(2, 2, 16, 64, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)
        P.store(x, range(16, 32), cache, scale)
        got = P.values(cache, scale)[1].transpose(0, 1)
        # half a step of 3 bits of mantissa, or of the smallest step of the block
        assert ((got - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0 ** -4, x.abs().max().double() * 2.0 ** -17)).all()


def test_a_page_filled_in_pieces_is_the_page_filled_at_once():
    """But for numbers below e4m3's normal range, which may be rounded twice: half a step more of the block's smallest."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(16, 2, 64, generator=g) * torch.exp2(torch.linspace(-6, 6, 16))[:, None, None]
    whole, parts = [(torch.zeros(1, 2, 16, 64, dtype=torch.uint8), torch.zeros(1, 2, dtype=torch.uint8)) for _ in range(2)]
    P.store(x, range(16), *whole)
    for t in range(16):
        P.store(x[t:t + 1], [t], *parts)
    assert torch.equal(whole[1], parts[1])
    a, b = P.values(*whole), P.values(*parts)
    unit = torch.exp2(whole[1].double() - 127)[..., None, None]
    assert ((a - b).abs() <= unit * 2.0 ** -9).all()
    normal = x.transpose(0, 1)[None].abs().double() >= unit * 2.0 ** -5
    assert torch.equal(a[normal], b[normal])


def test_the_engines_option(tmp_path):
    import argparse
    from redline_b200.apps.cli_common import add_engine_options, engine_options
    from redline_b200.config import EngineConfig
    assert EngineConfig.from_options("m", {}).torch_cache_dtype == torch.bfloat16
    assert EngineConfig.from_options("m", dict(dtype="float32")).torch_cache_dtype == torch.float32
    assert EngineConfig.from_options("m", dict(kv_cache_dtype="fp8")).torch_cache_dtype == kernels.KV8_DTYPE
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        EngineConfig.from_options("m", dict(kv_cache_dtype="int8"))
    ap = argparse.ArgumentParser()
    add_engine_options(ap)
    assert engine_options(ap.parse_args([]))["kv_cache_dtype"] == "auto"
    assert engine_options(ap.parse_args(["--kv-cache-dtype", "fp8"]))["kv_cache_dtype"] == "fp8"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_engines_pools(dtype):
    """A group in 8 bits beside one in the activations' type: types, shapes, starts on 16 bytes, no byte shared, sizes."""
    from redline_b200.cache.manager import GroupInfo
    from redline_b200.cache.storage import CacheStorage, bytes_per_page
    from redline_b200.parts.spec import CacheSpec
    groups = [GroupInfo(CacheSpec.keys_values_eight_bit("full", 3, 80), [0, 2, 5]), GroupInfo(CacheSpec.keys_values("full", 3, 80), [1])]
    assert groups[0].spec.typed() and not groups[1].spec.typed() and groups[0].spec.elements_per_token() == 2 * 3 * 80
    assert bytes_per_page(groups, 16, dtype.itemsize) == [3 * (2 * 3 * 80 * 16 + 2 * 3), 2 * 3 * 80 * 16 * dtype.itemsize]
    store = CacheStorage(groups, [7, 5], 16, dtype, torch.device("cpu"))
    spans = []
    for owner in (0, 2, 5):
        c = store.of_owner(owner, True)
        k, v, ks, vs = c.eight_bit
        assert k.dtype == v.dtype == kernels.KV8_DTYPE and ks.dtype == vs.dtype == kernels.KV8_SCALE_DTYPE
        assert k.shape == v.shape == (7, 3, 16, 80) and ks.shape == vs.shape == (7, 3) and c.group == 0
        for t in c.eight_bit:
            assert t.is_contiguous() and t.data_ptr() % 16 == 0 and not t.view(torch.uint8).any()
            spans.append((t.data_ptr(), t.data_ptr() + t.numel()))
    spans.sort()
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
    assert store.pools[0].data_ptr() <= spans[0][0] and spans[-1][1] <= store.pools[0].data_ptr() + store.pools[0].numel()
    plain = store.of_owner(1, True)
    assert plain.k.dtype == dtype and plain.k.shape == (5, 3, 16, 80)
    assert sum(b - a for a, b in spans) <= 7 * bytes_per_page(groups, 16, dtype.itemsize)[0] <= store.pools[0].numel()


def test_the_mixers_cache():
    from redline_b200.config import RopeScaling
    from redline_b200.parts import PartSpec, build_part
    from redline_b200.parts.attention import AttentionParams
    from redline_b200.parts.base import Runtime
    from redline_b200.parts.rope import RotaryParams
    position = PartSpec("rope", RotaryParams(16, 10000.0, RopeScaling(), 64))
    spec = PartSpec("gqa_attention", AttentionParams(64, 4, 2, 16, position, window=24))
    cpu = torch.device("cpu")
    plain = build_part("mixer", spec, Runtime(cpu, torch.bfloat16, 8, 2, 64, 16)).cache_spec()
    eight = build_part("mixer", spec, Runtime(cpu, torch.bfloat16, 8, 2, 64, 16, cache_dtype=kernels.KV8_DTYPE)).cache_spec()
    assert [(t.name, t.shape, t.dtype) for t in plain.tensors] == [("k", (2, 16), None), ("v", (2, 16), None)]
    assert [t.name for t in eight.tensors] == ["k", "v", "k_scale", "v_scale"] and (eight.kind, eight.window) == ("window", 24)
    assert plain.group_key() != eight.group_key()
