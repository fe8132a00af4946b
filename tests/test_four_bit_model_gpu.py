"""Models whose keys and values are kept in 4 bits, through the engine, against the plain implementations with keys and values rounded
the same way: whole prompts, single tokens through recorded steps, portions, mixed batches; the entry points; models that are refused."""
import io
import os
import subprocess
import sys

import numpy as np
import pytest

import four_bit as F
import girolorn_tiny
import plain_girolorn as PG
import plain_llama as PL
import tiny
import traces
from tiny import prompt_ids

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# fraction of the mean logit range (max, mean) that the engines are held to with 16- and 32-bit caches
TOL = {"float32": (2e-5, 2e-6), "bfloat16": (5e-2, 6e-3)}
# And what keys and values next to a border may add, as a share of what the rounding to 4 bits changes as a whole (max, mean).  In 32 bits hardly
# one number in a million lies so near a border that it takes the other side; one that does moves by one step.  Bfloat16's products are off by up
# to 2^-8 where steps are a fourth of a number: one code in fifty and, squares added up, a seventh of the rounding's effect, twice that with what
# the layers behind do to it.
BORDER = {"float32": (0.2, 0.01), "bfloat16": (1.0, 0.4)}


def four(x):
    return F.fast_rounded(np.asarray(x))[2]


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    """name -> (folder, vocabulary, requests, prompt lengths, logits with a 4-bit cache, logits with a 64-bit one)."""
    out = {}
    for name in ("A", "B", "D", "W", "X", "G6", "G7"):
        d = str(tmp_path_factory.mktemp("four" + name))
        lens, extra = ([3, 40, 64, 90], 24) if name not in "DX" else ([2, 130, 300], 24)
        if name.startswith("G"):
            girolorn_tiny.make_model(name, d)
            cfg, w = PL.load_folder(d)
            vocab, plain, place, attr = cfg["vocab"], lambda t: PG.forward(cfg, w, t), PG, "attend"
        else:
            if name in "WX":        # more heads over one key/value head than a block of rows holds; blocks whose key ranges a kernel of its own adds up
                from xyntetik_runner_amd.weights import write_random_model
                heads, dim = {"W": (21, 64), "X": (16, 128)}[name]
                write_random_model(dict(tiny.TINY_B, num_attention_heads=heads, num_key_value_heads=1, head_dim=dim), d, seed=7, std=0.05)
            else:
                tiny.make_model(name, d)
            cfg, w = PL.load_folder(d)
            vocab, plain, place, attr = cfg["vocab_size"], lambda t: PL.forward(cfg, w, t, all_at_once=True), PL, "attention_all_at_once"
        reqs = {f"r{i}": prompt_ids(n + extra, vocab, 1700 + i) for i, n in enumerate(lens)}
        exact = {rid: plain(t) for rid, t in reqs.items()}
        real = getattr(place, attr)
        setattr(place, attr, lambda q, k, v, *a, **kw: real(q, four(k), four(v), *a, **kw))
        try:
            rounded = {rid: plain(t) for rid, t in reqs.items()}
        finally:
            setattr(place, attr, real)
        out[name] = (d, vocab, reqs, {f"r{i}": n for i, n in enumerate(lens)}, rounded, exact)
    return out


def error(got, want):
    rng = float(np.mean(want.max(axis=-1) - want.min(axis=-1)))
    d = np.abs(np.asarray(got, dtype=np.float64) - want) / rng
    return float(d.max()), float(d.mean())


@pytest.mark.parametrize("schedule", ["whole", "tail", "portions", "mixed"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name,page", [("A", 16), ("B", 32), ("D", 64), ("W", 32), ("X", 32), ("G6", 8), ("G7", 64)])
def test_every_way_of_cutting(models, tmp_path, name, page, dtype, schedule):
    from xyntetik_runner_amd.engine.runner import ModelRunner
    from xyntetik_runner_amd.trace import replay
    d, vocab, reqs, plens, want, exact = models[name]
    steps = {"whole": lambda: traces.whole(reqs), "tail": lambda: traces.tail_one_by_one(reqs, tail=24), "portions": lambda: traces.portions(reqs),
             "mixed": lambda: traces.mixed(reqs, plens, max_live=3, seed=5)}[schedule]()
    runner = ModelRunner.from_folder(d, dtype=dtype, max_tokens=traces.max_live_tokens(steps, 64), page_size=page, max_requests=3, cache_dtype="mxfp4")
    for lc in runner.storage.layers:                    # old keys must never show: they start as NaN
        for pages in (lc.k, lc.v):
            pages.scales.fill_(255)
    out = str(tmp_path / "out")
    replay(runner, traces.to_lines(steps), out, report=io.StringIO())
    runner.manager.check()
    assert not runner.manager.requests and runner.manager.all_free()
    if schedule == "tail":
        assert runner.graphs.replays > 0
    got = traces.collect(steps, out, vocab)
    for rid in want:
        assert np.isfinite(got[rid]).all()
        most, mean = error(got[rid], want[rid])
        most4, mean4 = error(exact[rid], want[rid])     # what the rounding itself changes
        assert most <= TOL[dtype][0] + BORDER[dtype][0] * most4, (rid, most, most4)
        assert mean <= TOL[dtype][1] + BORDER[dtype][1] * mean4, (rid, mean, mean4)


def test_entry_points(models, tmp_path):
    """``LLM(cache_dtype=)``, the command line and the trace tool; a step run ahead, preemption, and a cache of more tokens in the same memory."""
    from xyntetik_runner_amd import LLM, SamplingParams
    d, vocab, reqs, plens, want, _ = models["B"]
    prompts = [reqs[r][:plens[r]] for r in reqs]
    greedy = SamplingParams(temperature=0.0, max_new_tokens=12, ignore_eos=True)
    roomy = LLM(d, dtype="bfloat16", max_tokens=1024, page_size=32, cache_dtype="mxfp4").generate(prompts, greedy)
    tight = LLM(d, dtype="bfloat16", max_tokens=160, page_size=32, cache_dtype="mxfp4")
    assert [len(t) for t in tight.generate(prompts, greedy)] == [12] * len(prompts) == [len(t) for t in roomy]
    tight.runner.manager.check()
    # one request alone: its first token is the plain implementation's where that is decided by more than rounding
    first = want["r3"][plens["r3"] - 1]
    two = np.sort(first)[-2:]
    if two[1] - two[0] > 0.1 * (first.max() - first.min()):
        assert roomy[3][0] == int(first.argmax())
    sixteen, four_ = (LLM(d, dtype="bfloat16", max_tokens=1024, page_size=32, cache_dtype=c).runner.storage.bytes_per_token() for c in ("auto", "mxfp4"))
    assert four_ * 16 == sixteen * 4.25
    cmd = [sys.executable, os.path.join(ROOT, "bin", "runner"), "-m", d, "--ids", ",".join(map(str, prompts[0])), "-n", "4", "--temp", "0", "--cache-dtype"]
    p = subprocess.run(cmd + ["mxfp4"], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0 and len(p.stdout.strip().split(",")) <= len(prompts[0]) + 4, p.stderr
    bad = subprocess.run(cmd + ["int3"], capture_output=True, text=True, timeout=120)
    assert bad.returncode == 1 and "expected auto" in bad.stderr


def test_models_that_are_refused(tmp_path):
    import kegorax_tiny
    import pevolorn_tiny
    import sugosun_tiny
    import suripel_tiny
    from xyntetik_runner_amd.engine.runner import ModelRunner
    for module, names in ((suripel_tiny, ["S1"]), (sugosun_tiny, ["G1"]), (kegorax_tiny, ["K1"]), (pevolorn_tiny, ["P1"]), (girolorn_tiny, ["G2"])):
        for name in names:      # (the last: heads of 10 and 14 channels)
            d = str(tmp_path / (module.__name__ + name))
            os.mkdir(d)
            module.make_model(name, d)
            with pytest.raises(ValueError, match="cache"):
                ModelRunner.from_folder(d, dtype="bfloat16", max_tokens=256, page_size=16, max_requests=2, cache_dtype="mxfp4")
    d = str(tmp_path / "A")
    os.mkdir(d)
    tiny.make_model("A", d)
    for bad in (dict(cache_dtype="fp8"), dict(cache_dtype="mxfp4", page_size=4)):
        with pytest.raises(ValueError):
            ModelRunner.from_folder(d, dtype="bfloat16", max_tokens=256, max_requests=2, **bad)
