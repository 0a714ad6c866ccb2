"""An engine whose cache holds keys and values in 8 bits, in a pool too small for all requests at once: the tokens that come out."""

import pytest

import tiny_configs as C
from gpu_utils import make_model, random_tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("kv8_preempted")
    return {n: make_model(tmp, C.ALL[n], seed=140 + i, sharpen=5.0)[0] for i, n in enumerate(C.ALL)}


@pytest.mark.parametrize("name", ["tiny_a", "tiny_b", "tiny_c"])
@pytest.mark.parametrize("graphs,ahead", [(True, True), (True, False), (False, True)])
def test_preempted_requests_give_the_tokens_that_others_give(name, graphs, ahead, models):
    """float32, greedy.  A preempted request's keys are computed anew in portions, where they were stored one by one before: the same scales, and
    the same numbers but for those below e4m3's normal range, twice rounded: 2^-18 of a block's largest.  That moves hidden states by some 2^-17
    of themselves and logits, a hundred or so, by less than 2^-9 in a few layers: logarithms of probabilities by less than 1e-2."""
    from redline_b200.engine.engine import Engine
    V = C.ALL[name]["vocab_size"]
    prompts = [random_tokens(V, n, 90 + n) for n in (40, 35, 44, 38, 63)]

    def run(**kw):
        opts = dict(dtype="float32", kv_cache_dtype="fp8", max_num_seqs=5, max_num_batched_tokens=64, max_seq_len=128, kv_cache_tokens=1024,
                    async_scheduling=False, cuda_graphs=False)
        opts.update(kw)
        eng = Engine(models[name], **opts)
        outs = eng.generate(prompts, max_new_tokens=24, ignore_eos=True)
        eng.runner.check_status()
        return eng, outs

    _, want = run()
    small, got = run(kv_cache_tokens=192, admission_watermark=0.0, async_scheduling=ahead, cuda_graphs=graphs)
    assert small.num_preemptions > 0 and small.runner.cache.num_open() == 0
    for a, b in zip(got, want):
        assert a["output_ids"] == b["output_ids"]
        assert all(abs(x - y) < 1e-2 for x, y in zip(a["logprobs"], b["logprobs"]))
