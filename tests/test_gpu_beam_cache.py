"""PagedCache and BeamSearch (p0pc0rn_b200.beam) around their steps: what they report of shortages, after compacting and
after later steps, on small caches and models."""
import numpy as np
import pytest

from p0pc0rn_b200 import beam

from . import kv_ref as R
from .test_gpu_beam_search import CFG, rope_table
from .test_gpu_decode_step import host_model, upload_model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(g):
    h = host_model(CFG, 901)
    h["rope"] = {k: rope_table(160, CFG["hd"] // 2, 79 + i) for i, k in enumerate(("full", "sliding"))}
    return upload_model(g, h)


def test_a_cache_reports_short_steps(g, monkeypatch):
    parents = lambda *p: {"buf": g.upload(np.array(p, np.uint32))}
    monkeypatch.setattr(beam, "LOG", 8)
    c = beam.PagedCache(g, 2, 1, 1, 64, 2, 4)
    assert c.short() == 0 and c.ran_short() == 0
    c.step(add=64)                                                   # both pages
    assert c.short() == 0 and c.ran_short() == 0
    c.compact()
    assert c.short() == 0 and c.ran_short() == 0                     # two pages in use are no shortage
    c.step(add=1)
    assert c.short() == 2
    c.step(parent=parents(0, R.NONE), add=1)                         # one row goes, the other has its page
    assert c.short() == 0 and c.ran_short() == 2
    for _ in range(20):                                              # more steps than the record holds
        c.step(parent=parents(0, R.NONE), add=0)
    assert c.short() == 0 and c.ran_short() == 2


def test_result_after_compacting(g, model):
    s = beam.BeamSearch(g, CFG, model, 160)
    s.prompt([3, 1400, 77])
    for _ in range(3):
        s.step()
    want = s.result()
    for cache in s.cache.values():
        cache.compact()
    got = s.result()
    assert got[0] == want[0] and np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    g.done()
    s.close()


def test_result_refuses_after_a_shortage(g, model):
    # the first fork finds no pages; a step after pages were given back succeeds, but the hypotheses are not the search's any more
    s = beam.BeamSearch(g, CFG, model, 160, spare_pages=1 - CFG["beams"] * 3)
    s.prompt([3, 1400, 77])
    assert s.result()[0]
    s.step()
    for cache in s.cache.values():
        assert cache.short() == CFG["beams"] - 1
        cache.step(parent={"buf": g.upload(np.array([0] + [R.NONE] * 3, np.uint32))}, add=0)
        assert cache.short() == 0
    with pytest.raises(RuntimeError, match="short of %d pages" % (CFG["beams"] - 1)):
        s.result()
    g.done()
    s.close()


def test_close_gives_the_memory_back(g, model):
    before, held = g.stats["alive"], len(g.bufs)
    s = beam.BeamSearch(g, CFG, model, 160)
    s.prompt([3])
    s.step()
    s.close()
    tables = sum(b.size for c in s.cache.values() for st in c.state for b in st.values())
    assert g.stats["alive"] - before == tables                       # the caches' states can still be read
    for c in s.cache.values():
        assert g.read(c.state[c.now]["len"], 0, 4, np.uint32)[0] == 2
        c.close()
    assert g.stats["alive"] == before and len(g.bufs) == held
    s.close()                                                        # again: nothing left to do


def test_prompts_that_are_refused(g, model):
    # without a token there is nothing to select from; a second prompt would write over the rows' last tokens
    s = beam.BeamSearch(g, CFG, model, 160)
    for tokens in ([], [5] * 161):
        with pytest.raises(ValueError, match="a prompt of %d tokens" % len(tokens)):
            s.prompt(tokens)
    s.prompt([3, 9])
    want = s.result()
    with pytest.raises(ValueError, match="has its prompt"):
        s.prompt([4])
    got = s.result()
    assert got[0] == want[0] and np.array_equal(got[1], want[1])
    g.done()
    s.close()
