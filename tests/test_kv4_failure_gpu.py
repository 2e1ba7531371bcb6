"""What the attention over the 4-bit cache does when a wait inside it runs out,
without a GPU fault: every wait is bounded (2 s), the test aid
g4_test_kv4_attention_starve makes those of the first CTA run out (a copy that
is never issued, a tile that is never announced, a wait that counts as run out),
and the rows of that CTA become NaN, in all dimensions; the others keep their
bits, and the next call is what it always was."""
import time

import numpy as np
import pytest

from test_kv4_gpu import Setup, check_attention

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def starved(g4, s, q, what):
    out = torch.full_like(q, 5)
    ws = torch.empty(g4.kv4_attention_workspace(s.cache, s.batch, 0, q.shape[1]), dtype=torch.uint8, device="cuda:0")
    assert g4.load().g4_test_kv4_attention_starve(what) == 0
    t = time.time()
    s.attend(q, out, 0, 0.1, 0, ws=ws)
    torch.cuda.synchronize()
    return out, time.time() - t


def check_starved(g4, s, q, want, what, rows):
    got, took = starved(g4, s, q, what)
    assert took < 20, took                              # a few waits of 2 s, one after the other
    bad = torch.zeros(len(got), dtype=torch.bool)
    bad[rows] = True
    assert torch.isnan(got[bad]).all()
    assert torch.equal(got[~bad], want[~bad])
    again = torch.empty_like(q)
    s.attend(q, again, 0, 0.1, 0)
    assert torch.equal(again, want)


@pytest.mark.parametrize("hd", [256, 512])
def test_few_rows(g4, hd):
    """A copy that is never issued: the first CTA works on the first sequence."""
    s = Setup(g4, [(3000, 1), (40, 1), (700, 2)], 1, hd, 64)
    q, want = check_attention(g4, s, 8, "f32", 0.1, 0, np.random.default_rng(hd))
    check_starved(g4, s, q, want, 1, [0])


@pytest.mark.parametrize("what", [1, 2])
@pytest.mark.parametrize("hd", [256, 512])
@pytest.mark.parametrize("start", [0, 1200])
def test_many_rows(g4, start, hd, what):
    """K that is never announced, and a conversion warp that gave up while the rest went on: the
    first CTA works on the last row tile (16 tokens of 8 heads), for 512 dimensions in a pair
    whose halves of the scores reach each other."""
    s = Setup(g4, [(start, 200)], 1, hd, 64)
    q, want = check_attention(g4, s, 8, "f32", 0.1, 0, np.random.default_rng(hd))
    check_starved(g4, s, q, want, what, slice(192, 200))


def test_refused_where_there_is_no_such_kernel(g4):
    s = Setup(g4, [(0, 200)], 1, 64, 64)
    q, want = check_attention(g4, s, 8, "f32", 0.1, 0, np.random.default_rng(1))
    assert g4.load().g4_test_kv4_attention_starve(3) == -1
    assert g4.load().g4_test_kv4_attention_starve(1) == 0
    out = torch.full_like(q, 5)
    with pytest.raises(g4.G4Error):
        s.attend(q, out, 0, 0.1, 0)
    s.attend(q, out, 0, 0.1, 0)
    assert torch.equal(out, want)
