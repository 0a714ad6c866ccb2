"""An engine whose cache holds keys and values in 8 bits: what every attention layer stores and puts out in every step against the
restatement (plain_kv8.py, the tolerances of test_kv8_gpu.py), the ways an engine runs its steps, pages that change hands, refusals."""

import math

import pytest
import torch

import kapitar_configs
import kapitar_utils
import plain_kv8 as P
import tiny_configs as C
from gpu_utils import make_model, random_tokens
from test_kv8_gpu import near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("kv8_models")
    return {n: make_model(tmp, C.ALL[n], seed=140 + i, sharpen=5.0)[0] for i, n in enumerate(C.ALL)}


class Watch:
    """Wraps ``GQAttention._attend``: the stored bytes bit for bit, the outputs against attention in float64."""

    def __init__(self, monkeypatch, dtype):
        from redline_b200.parts.attention import GQAttention
        self.kept, self.dtype, self.calls, self.fused = {}, dtype, 0, 0
        plain = GQAttention._attend

        def attend(mixer, qkv, ctx, cache):
            before = qkv.clone()
            out = plain(mixer, qkv, ctx, cache)
            self.check(mixer, before, qkv, ctx, cache, out)
            return out

        monkeypatch.setattr(GQAttention, "_attend", attend)

    def check(self, mixer, before, after, ctx, cache, out):
        p, T = mixer.params, ctx.T
        heads, kv_heads, dim, page = p.num_heads, p.num_kv_heads, p.head_dim, mixer.rt.page_size
        held = cache.eight_bit
        if cache.k.data_ptr() not in self.kept:
            self.kept[cache.k.data_ptr()] = [torch.zeros(t.shape, dtype=torch.uint8) for t in held]
        mine = self.kept[cache.k.data_ptr()]
        cos, sin = (t.cpu() for t in mixer.position.rotary_tables())
        at = ctx.positions.cpu().long()[:T]
        g = ctx.groups[cache.group]
        table, slots = g.block_table.cpu(), g.slots.cpu()[:T]
        q, k, v = before.cpu().float().split([heads * dim, kv_heads * dim, kv_heads * dim], -1)
        P.store(P.rotate(k.view(T, kv_heads, dim), cos[at], sin[at]), slots, mine[0], mine[2])
        P.store(v.reshape(T, kv_heads, dim), slots, mine[1], mine[3])
        for got, want in zip(held, mine):
            assert torch.equal(got.view(torch.uint8).cpu(), want)
        q = P.rotate(q.view(T, heads, dim), cos[at], sin[at])
        if not torch.equal(before, after):             # (rotated on its way into the cache: rounded)
            q = after[:, :heads * dim].cpu().view(T, heads, dim)
        elif at.max() > 0:
            self.fused += 1
        keys, vals = P.values(mine[0], mine[2]), P.values(mine[1], mine[3])
        for s, (first, n, start) in enumerate(zip(ctx.host.q_start, ctx.host.q_len, ctx.host.start_pos)):
            ref = P.attend(q[first:first + n], keys, vals, table[s], range(start, start + n), p.window, mixer.scale)
            near(out[first:first + n].view(n, heads, dim), ref, vals[table[s][:-(-(start + n) // page)].long()], self.dtype)
        self.calls += 1


@pytest.mark.parametrize("name,dtype,page", [("tiny_a", "bfloat16", 16), ("tiny_b", "bfloat16", 32), ("tiny_b", "bfloat16", 64),
                                             ("tiny_a", "float32", 16), ("tiny_c", "bfloat16", 16)])
def test_every_layer_of_every_step(name, dtype, page, models, monkeypatch):
    """Prompts in portions beside single tokens, single tokens together, pages that a second batch of requests takes over."""
    from redline_b200.engine.engine import Engine
    eng = Engine(models[name], dtype=dtype, kv_cache_dtype="fp8", max_num_seqs=3, max_num_batched_tokens=48, max_seq_len=192,
                 kv_cache_tokens=448, cuda_graphs=False, async_scheduling=False, block_size=page)
    watch = Watch(monkeypatch, dtype)
    V = C.ALL[name]["vocab_size"]
    for batch in ((5, 70, 33, 100), (50, 1)):
        outs = eng.generate([random_tokens(V, n, 7 + n) for n in batch], max_new_tokens=9, ignore_eos=True)
        assert all(len(o["output_ids"]) == 9 for o in outs)
    assert len(eng.score(random_tokens(V, 90, 3))) == 89
    assert watch.calls > 40 and watch.fused > 0
    eng.runner.check_status()


@pytest.mark.parametrize("name,dtype", [("tiny_a", "float32"), ("tiny_c", "float32"), ("tiny_a", "bfloat16"), ("tiny_b", "bfloat16")])
def test_graphs_and_preemption(name, dtype, models):
    """Steps replayed as graphs give the tokens that eager steps give (float32; in bfloat16 the padding rows may turn sums around), a
    pool too small for all requests at once included; logarithms of probabilities are finite; the cache takes about half the memory."""
    from redline_b200.engine.engine import Engine
    V = C.ALL[name]["vocab_size"]
    prompts = [random_tokens(V, n, 90 + n) for n in (40, 35, 44, 38, 63)]

    def run(**kw):
        opts = dict(dtype=dtype, kv_cache_dtype="fp8", max_num_seqs=5, max_num_batched_tokens=64, max_seq_len=128,
                    kv_cache_tokens=1024, async_scheduling=False)
        opts.update(kw)
        eng = Engine(models[name], **opts)
        outs = eng.generate(prompts, max_new_tokens=24, ignore_eos=True)
        eng.runner.check_status()
        assert all(math.isfinite(x) for o in outs for x in o["logprobs"])
        return eng, [o["output_ids"] for o in outs]

    eager, want = run(cuda_graphs=False)
    graphs, got = run()
    assert graphs.runner.num_graph_steps > 0 and eager.runner.num_graph_steps == 0
    if dtype == "float32":
        assert got == want
    assert graphs.describe()["config"]["kv_cache_dtype"] == "fp8"
    full, _ = run(kv_cache_dtype="auto")
    ratio = graphs.memory_report()["kv_cache"] / full.memory_report()["kv_cache"]
    assert ratio < (0.3 if dtype == "float32" else 0.53)
    small, _ = run(kv_cache_tokens=192, admission_watermark=0.0, async_scheduling=True)
    assert small.num_preemptions > 0 and small.runner.cache.num_open() == 0


def test_refusals(models, tmp_path):
    from redline_b200.engine.engine import Engine
    from redline_b200.engine.runner import EngineError
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        Engine(models["tiny_a"], kv_cache_dtype="int4")
    d, _ = kapitar_utils.make_model(tmp_path, kapitar_configs.ATTN, seed=3)
    with pytest.raises(EngineError, match="bfloat16 only"):
        Engine(d, dtype="bfloat16", kv_cache_dtype="fp8", max_num_seqs=2, max_num_batched_tokens=64, max_seq_len=64, kv_cache_tokens=128)
