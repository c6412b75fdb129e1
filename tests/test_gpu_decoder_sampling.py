"""Sampled generation of the LUT decoder: every token is the one that sample_tokens and the fp64 oracle
draw from the step's logits with the step's number, one step at a time, in one call and from a captured
step; settings change between replays; greedy generation beside it keeps its tokens."""
import numpy as np
import pytest

from oracle import kve

pytestmark = pytest.mark.gpu

SMALL = dict(hidden=256, layers=2, q_heads=4, kv_heads=2, intermediate=384, vocab=1000,
             max_context=96, page_size=16, max_steps=8)
CONTEXT = 20


@pytest.fixture(scope="module")
def dec(pkg):
    return pkg.decoder


@pytest.fixture
def made(dec, dev):
    d, weights = dec.synthetic_decoder(dec.DecoderConfig(**SMALL), context=CONTEXT, seed=5, device=dev,
                                       keep_weights=True)

    def start():
        for i, w in enumerate(weights["layers"]):
            d.set_context(i, w["k_codes"], w["k_scales"], w["v_codes"], w["v_scales"], CONTEXT)
        d.reset(CONTEXT)
    yield d, start
    d.close()


def numbers(n, seed):
    return np.random.default_rng(seed).uniform(size=n).astype(np.float32)


SETTINGS = [dict(), dict(temperature=0.7, top_k=40, top_p=0.9, min_p=0.05), dict(temperature=2.5, top_p=0.5),
            dict(top_k=3), dict(min_p=0.2), dict(temperature=0.0), dict(temperature=30.0, top_k=1000)]


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
def test_steps_call_and_graph_agree(dec, dev, made, settings):
    import torch
    d, start = made
    n, u = 4, numbers(4, 3)
    start()
    token, steps = 7, []
    for i in range(n):
        toks, logits = d.generate(token, 1, use_graph=False, return_logits=True, uniform=u[i:i + 1], **settings)
        full = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) | settings
        rows = {k: torch.tensor([v], dtype=torch.int32 if k == "top_k" else torch.float32, device=dev)
                for k, v in full.items()}
        got = dec.sample_tokens(torch.tensor(logits, device=dev)[None], torch.tensor(u[i:i + 1], device=dev), **rows)
        assert int(toks[0]) == int(got[0]), i
        f = lambda k: float(np.float32(full[k]))  # noqa: E731
        assert int(toks[0]) == kve.draw(logits, float(u[i]), f("temperature"), full["top_k"], f("top_p"), f("min_p"))
        if settings.get("temperature") == 0.0:
            assert int(toks[0]) == int(np.argmax(logits))
        token = int(toks[0])
        steps.append(token)
    for use_graph in (False, True, True):
        start()
        toks, last = d.generate(7, n, use_graph=use_graph, return_logits=True, uniform=torch.tensor(u), **settings)
        assert toks.tolist() == steps, use_graph
        assert np.array_equal(last, logits)


def test_one_captured_step_follows_settings_and_numbers(dec, made):
    """Greedy and sampled generations alternate on one decoder, each with its captured step."""
    d, start = made
    start()
    greedy = d.generate(7, 6, use_graph=False).tolist()
    want = []
    for i, s in enumerate(SETTINGS):
        start()
        want.append(d.generate(7, 6, use_graph=False, uniform=numbers(6, i), **s).tolist())
    assert len({tuple(w) for w in want}) > 3 and want[5] == greedy
    for _ in range(2):
        for i, s in enumerate(SETTINGS):
            start()
            assert d.generate(7, 6, uniform=numbers(6, i), **s).tolist() == want[i], s
            start()
            assert d.generate(7, 6).tolist() == greedy
    # as many steps as fit, then one
    start()
    assert d.generate(7, 8, uniform=numbers(8, 1), **SETTINGS[1]).shape == (8,)
    assert d.generate(7, 1, uniform=numbers(1, 1), **SETTINGS[1]).shape == (1,)


def test_logits_without_a_distribution(dec, made):
    d, start = made
    c = d.cfg
    lm = dec._linear(np.random.default_rng(1), c.vocab, c.hidden, 0.05, 0.0038, 0.05, False)[0]
    norm = np.ones(c.hidden, np.float32)
    norm[3] = np.nan
    d.set_head(lm, norm, np.ones((c.vocab, c.hidden), np.float32))
    for use_graph in (False, True):
        start()
        toks, logits = d.generate(7, 4, use_graph=use_graph, return_logits=True, uniform=numbers(4, 2))
        assert np.isnan(logits).all() and toks.tolist() == [-1] * 4
    start()
    assert d.generate(7, 3, use_graph=False).tolist() == [0, 0, 0]


def test_refusals_change_nothing(pkg, dec, made):
    d, start = made
    u = numbers(4, 0)
    start()
    want = d.generate(7, 4, use_graph=False, uniform=u).tolist()
    start()
    for bad in (np.nan, -0.25, 1.0, np.inf):
        with pytest.raises(pkg.OjasxError, match="uniform"):
            d.generate(7, 4, uniform=np.where(np.arange(4) == 3, bad, u))
    for s in (dict(temperature=-1.0), dict(temperature=np.nan), dict(temperature=np.inf), dict(top_p=-0.1),
              dict(top_p=np.nan), dict(min_p=1.5), dict(min_p=-0.1)):
        with pytest.raises(pkg.OjasxError, match="sampling"):
            d.generate(7, 4, uniform=u, **s)
    with pytest.raises(pkg.OjasxError, match="max_steps"):
        d.generate(7, 9, uniform=numbers(9, 0))
    with pytest.raises(ValueError, match="uniform"):
        d.generate(7, 4, uniform=u[:3])
    with pytest.raises(ValueError, match="uniform"):
        d.generate(7, 4, temperature=0.5)
    # the largest number below 1, also where float32 would round it up
    assert d.generate(7, 4, use_graph=False, uniform=u).tolist() == want
    start()
    assert d.generate(7, 1, uniform=[1 - 2.0 ** -30]).tolist()[0] >= 0
