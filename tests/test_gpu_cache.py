"""Engines whose talker cache is kept in 4 bits or seen through a window, and
takes of one prompt, against the CPU oracle with the same cache.

The oracle's talker stack is given the cache's rounding (bf16, or the 4-bit form
in float64) and mask. Bounds are those of the other parity tests: logits within
2e-2, greedy codes equal wherever the oracle's top-2 gap exceeds 1e-2. A 4-bit
code whose quotient lies within the projections' error (about 1e-5 of a step)
of a border may fall on the other side: it moves one key entry by a step, at
most 3.2 / 7 for a unit-rms row, one score by 3 * 0.46 * 128 ** -0.5 = 0.12, that
key's weight of about 1 / 25 by 12 %, and a logit of these models by about
2e-3; a few of them stay within the bound."""
import numpy as np
import pytest
import torch

from oracle import kv as K
from oracle import qtts_oracle as O
from parity import check_codes

pytestmark = pytest.mark.gpu

LOGIT_TOL = 2e-2
GREEDY = O.SamplingConfig(False, 0, 1.0, 1.0)
SAMPLED = O.SamplingConfig(True, 50, 1.0, 0.9)
CACHES = [(16, 8, 2), (16, 1, 0), (4, 0, 0), (4, 12, 3)]


class CacheStack(O.DecoderStack):
    """The decoder stack with a rounded cache and a mask of its own."""

    bits, window, sinks = 16, 0, 0

    def held(self, x):
        if self.bits == 16:
            return x.to(torch.bfloat16).float()
        return torch.from_numpy(K.quantise_fast(x.numpy())).float()

    def _layer(self, li, x, offset):
        d, L = self.d, self.layers[li]
        S = x.shape[0]
        normed = O.rmsnorm(x, L["in_g"], d.eps)
        q, k, v = ((normed @ L[n].T).view(S, -1, d.head_dim) for n in "qkv")
        cos, sin = O.rope_tables(d.theta, d.head_dim, np.arange(offset, offset + S))
        q = O.rope(O.rmsnorm(q, L["q_g"], d.eps), cos, sin)
        k = O.rope(O.rmsnorm(k, L["k_g"], d.eps), cos, sin)
        self.k_cache[li][:, offset:offset + S] = self.held(k.contiguous()).transpose(0, 1)
        self.v_cache[li][:, offset:offset + S] = self.held(v.contiguous()).transpose(0, 1)
        T = offset + S
        kv_of_q = torch.arange(d.q_heads) // (d.q_heads // d.kv_heads)
        scores = torch.einsum("shd,htd->hst", q, self.k_cache[li][kv_of_q, :T]) / d.head_dim ** 0.5
        seen = torch.tensor([[K.sees(offset + s, t, self.window, self.sinks) for t in range(T)]
                             for s in range(S)])
        probs = torch.softmax(scores.masked_fill(~seen, -float("inf")), dim=-1)
        att = torch.einsum("hst,htd->shd", probs, self.v_cache[li][kv_of_q, :T]).reshape(S, -1)
        h1 = x + att @ L["o"].T
        post = O.rmsnorm(h1, L["post_g"], d.eps)
        gate = post @ L["gate"].T
        return h1 + (gate / (1.0 + torch.exp(-gate)) * (post @ L["up"].T)) @ L["down"].T


def oracle_with(model_dir, cache, steps=128):
    m = O.OracleModel(model_dir, steps)
    m.talker.__class__ = CacheStack
    m.talker.bits, m.talker.window, m.talker.sinks = cache
    return m


@pytest.fixture(scope="module")
def engine_of(pkg, model_dirs):
    made = {}

    def get(shape, cache):
        if (shape, cache) not in made:
            made[shape, cache] = pkg.HipTtsEngine.load_with_options(
                model_dirs[shape], pkg.EngineOptions(0, 128, *cache))
        return made[shape, cache]

    yield get
    for e in made.values():
        e.close()


def greedy(pkg, frames):
    return pkg.GenerateOptions(decode_audio=False, do_sample=False, subtalker_dosample=False,
                               repetition_penalty=1.0, max_frames=frames)


@pytest.mark.parametrize("shape", ["tiny", "tiny_proj"])
@pytest.mark.parametrize("cache", CACHES)
def test_prefill_and_steps(engine_of, model_dirs, shape, cache):
    e, m = engine_of(shape, cache), oracle_with(model_dirs[shape], cache)
    pre, _, _ = m.prepare(list(np.random.default_rng(2).integers(0, 4000, 31)))
    hidden, logits, _ = e.talker_prefill(pre.numpy())
    _, rh, rl = m.talker_prefill(pre)
    assert np.abs(hidden - rh.numpy()).max() <= LOGIT_TOL
    assert np.abs(logits - rl).max() <= LOGIT_TOL
    rng = np.random.default_rng(5)
    for off in range(pre.shape[0], pre.shape[0] + 4):
        x = rng.standard_normal(e.hidden).astype(np.float32) * 0.05
        h, l, t = e.talker_decode_step(x, off)
        _, rh, rl = m.talker_step(torch.from_numpy(x), off)
        print(f"[cache] {shape} {cache} at {off}: logits off by {np.abs(l - rl).max():.1e}")
        assert np.abs(l - rl).max() <= LOGIT_TOL and np.abs(h - rh.numpy()).max() <= LOGIT_TOL
        # the allocation-free step computes the same
        h2, l2, t2 = e.talker_decode_step_static(x, off)
        assert np.array_equal(l, l2) and np.array_equal(h, h2) and t == t2


@pytest.mark.parametrize("cache", CACHES)
def test_greedy_codes(engine_of, pkg, model_dirs, cache):
    e, m = engine_of("tiny", cache), oracle_with(model_dirs["tiny"], cache)
    ids = np.random.default_rng(3).integers(0, 4000, 12)
    out = e.generate_codes_from_ids(ids, greedy(pkg, 24))
    pre, tr, pad = m.prepare(list(ids))
    codes, _, recs = m.rollout(pre, tr, pad, 24, GREEDY, GREEDY, forced_codes=out.codes)
    check_codes(out.codes, codes, recs, f"cache {cache}")
    # repeated, and as a stream in chunks: the same codes
    assert e.generate_codes_from_ids(ids, greedy(pkg, 24)).codes == out.codes
    s = e.start_stream_from_ids(ids, greedy(pkg, 24), pkg.StreamOptions(text_lookahead_tokens=12))
    got = []
    while (c := s.next_codes_chunk(7)) is not None:
        got += c.codes
    assert got == out.codes
    s.close()


@pytest.mark.parametrize("cache", [(4, 0, 0), (16, 9, 4)])
def test_batch(engine_of, pkg, model_dirs, cache):
    e, m = engine_of("tiny", cache), oracle_with(model_dirs["tiny"], cache)
    reqs = [np.random.default_rng(s).integers(0, 4000, n) for s, n in enumerate((5, 23, 40))]
    outs = e.generate_codes_batch_from_ids(reqs, [greedy(pkg, 10)] * 3)
    for ids, out in zip(reqs, outs):
        pre, tr, pad = m.prepare(list(ids))
        codes, _, recs = m.rollout(pre, tr, pad, 10, GREEDY, GREEDY, forced_codes=out.codes)
        check_codes(out.codes, codes, recs, f"batch {cache}")


def test_window_wider_than_the_speech(engine_of, model_dirs):
    """A window that hides nothing gives the plain engine's logits (two kernels
    over the same bf16 rows: fp32 rounding apart)."""
    a, b = engine_of("tiny", (16, 0, 0)), engine_of("tiny", (16, 4096, 0))
    m = O.OracleModel(model_dirs["tiny"], 128)
    pre, _, _ = m.prepare(list(np.random.default_rng(7).integers(0, 4000, 50)))
    la, lb = a.talker_prefill(pre.numpy())[1], b.talker_prefill(pre.numpy())[1]
    assert np.abs(la - lb).max() <= 1e-3
    x = np.random.default_rng(8).standard_normal(a.hidden).astype(np.float32) * 0.05
    la, lb = (e.talker_decode_step(x, pre.shape[0])[1] for e in (a, b))
    assert np.abs(la - lb).max() <= 1e-3


@pytest.mark.parametrize("cache", [(16, 0, 0), (4, 0, 0), (16, 20, 2)])
@pytest.mark.parametrize("n_ids", [7, 23, 55])  # prompts of 16, 32 (a whole page) and 64 positions
def test_takes_equal_a_batch(engine_of, pkg, cache, n_ids):
    e = engine_of("tiny", cache)
    ids = np.random.default_rng(n_ids).integers(0, 4000, n_ids)
    opt = pkg.GenerateOptions(decode_audio=False, max_frames=20, rng="philox")
    seeds = [11, 5, 2 ** 63 + 7, 11, 0]
    takes = e.generate_codes_takes_from_ids(ids, seeds, opt)
    batch = e.generate_codes_batch_from_ids(
        [ids] * len(seeds), [pkg.GenerateOptions(decode_audio=False, max_frames=20, rng="philox",
                                                 seed=s) for s in seeds])
    assert [t.codes for t in takes] == [b.codes for b in batch]
    assert [t.ended_by_eos for t in takes] == [b.ended_by_eos for b in batch]
    assert takes[0].codes == takes[3].codes and takes[0].codes != takes[1].codes
    # again, fewer, and between other generations
    one = e.generate_codes_from_ids(ids, greedy(pkg, 6))
    assert [t.codes for t in e.generate_codes_takes_from_ids(ids, seeds[1:3], opt)] == \
        [b.codes for b in batch[1:3]]
    assert e.generate_codes_from_ids(ids, greedy(pkg, 6)).codes == one.codes
    assert [t.codes for t in e.generate_codes_batch_from_ids([ids], [greedy(pkg, 6)])] == \
        [t.codes for t in e.generate_codes_takes_from_ids(ids, [9], greedy(pkg, 6))]


def test_sixteen_takes_draw_as_the_oracle(engine_of, pkg, oracles):
    e, m = engine_of("tiny_proj", (16, 0, 0)), oracles["tiny_proj"]
    ids = np.random.default_rng(4).integers(0, 4000, 18)
    opt = pkg.GenerateOptions(decode_audio=False, max_frames=5)
    outs = e.generate_codes_takes_from_ids(ids, list(range(16)), opt)
    pre, tr, pad = m.prepare(list(ids))
    for seed, out in enumerate(outs):
        codes, _, recs = m.rollout(pre, tr, pad, 5, SAMPLED, SAMPLED, penalty=1.05, seed=seed,
                                   forced_codes=out.codes)
        check_codes(out.codes, codes, recs, f"take {seed}", sampled=True)


def test_takes_refusals(engine_of, pkg):
    e = engine_of("tiny", (16, 0, 0))
    opt = greedy(pkg, 4)
    for seeds in ([], list(range(17))):
        with pytest.raises(pkg.InvalidInput, match="takes"):
            e.generate_codes_takes_from_ids([1, 2, 3], seeds, opt)
    with pytest.raises(pkg.InvalidInput, match="cache steps"):
        e.generate_codes_takes_from_ids([1, 2, 3], [1], greedy(pkg, 500))
    with pytest.raises(pkg.InvalidInput, match="out of range"):
        e.generate_codes_takes_from_ids([10 ** 6], [1], opt)
    stream = e.start_stream_from_ids([1, 2, 3], opt)
    e.generate_codes_takes_from_ids([1, 2, 3], [1], opt)
    with pytest.raises(pkg.InvalidInput, match="superseded"):
        stream.next_codes_chunk(1)
    stream.close()


def test_full_size_cache(pkg, full_model_dir):
    """0.6B shapes, 4 bits and a window: a step's logits against the oracle, and
    takes against a batch."""
    d = full_model_dir("0.6b")
    cache = (4, 64, 9)
    e = pkg.HipTtsEngine.load_with_options(d, pkg.EngineOptions(0, 256, *cache))
    plain = pkg.HipTtsEngine.load_with_options(d, pkg.EngineOptions(0, 256))
    m = oracle_with(d, cache, 256)
    ids = np.random.default_rng(31).integers(0, 150000, 100)
    pre, _, _ = m.prepare(list(ids))
    _, logits, _ = e.talker_prefill(pre.numpy())
    _, _, rl = m.talker_prefill(pre)
    assert np.abs(logits - rl).max() <= 5 * LOGIT_TOL  # 28 layers and 16 heads: more codes near a border
    opt = pkg.GenerateOptions(decode_audio=False, max_frames=6, rng="philox")
    for eng in (e, plain):
        takes = eng.generate_codes_takes_from_ids(ids, [1, 2, 3], opt)
        batch = eng.generate_codes_batch_from_ids(
            [ids] * 3, [pkg.GenerateOptions(decode_audio=False, max_frames=6, rng="philox", seed=s)
                        for s in (1, 2, 3)])
        assert [t.codes for t in takes] == [b.codes for b in batch]
    # 72 bytes a row instead of 256
    rows = 28 * 2 * 8 * 256
    assert plain.info.device_bytes - e.info.device_bytes > 0.9 * rows * 184
    e.close()
    plain.close()
