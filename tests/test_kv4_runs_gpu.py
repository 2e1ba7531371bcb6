"""Prompt attention over the 4-bit cache where its output is summed up in memory
(more than 16 key tiles of 64 in a key range for fp32, more than 256 for 16-bit
types), and the calls near the bound between its two kernels. Which kernel a
call takes, and into how many key ranges it cuts a row tile, is read from the
launches that it makes (captured into a graph). Rows are compared with the
definition in 64 bits within the bound that kv4_ref.tolerance derives."""
import numpy as np
import pytest

import kv4_ref as ref
from test_kv4_gpu import Setup, TYPES, as64, check_attention, dev, kind_of, tensors

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def launches(call):
    """(kernel, blocks, threads) of each launch that `call(stream)` makes."""
    cu = pytest.importorskip("cuda.bindings.driver")

    def ok(r):
        assert int(r[0]) == 0, r
        return r[1] if len(r) == 2 else r[1:]
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        call(torch.cuda.current_stream().cuda_stream)
    g = cu.CUgraph(graph.raw_cuda_graph())
    n = ok(cu.cuGraphGetNodes(g, 0))[1]
    found = []
    for node in ok(cu.cuGraphGetNodes(g, n))[0]:
        if ok(cu.cuGraphNodeGetType(node)) != cu.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            continue
        p = ok(cu.cuGraphKernelNodeGetParams(node))
        name = ok(cu.cuFuncGetName(p.func)) if int(p.func) else ok(cu.cuKernelGetName(p.kern))
        found.append((name.decode(), p.gridDimX, p.blockDimX))
    return found


def ranges_of(g4, s, heads, name, window=0):
    """Key ranges of a row tile where the call takes the large tiles, 0 where it takes the small ones."""
    q = torch.zeros((s.rows, heads, s.hd), dtype=TYPES[name], device="cuda:0")
    out = torch.empty_like(q)
    ws = torch.empty(g4.kv4_attention_workspace(s.cache, s.batch, kind_of(g4, name), heads), dtype=torch.uint8,
                     device="cuda:0")
    s.attend(q, out, kind_of(g4, name), 0.1, window, ws=ws)        # what it sets up once is not part of a graph
    torch.cuda.synchronize()
    got = launches(lambda st: s.attend(q, out, kind_of(g4, name), 0.1, window, ws=ws, stream=st))
    torch.cuda.synchronize()
    if "k_kv4_prompt" not in got[0][0]:
        assert "k_kv4_attn" in got[0][0]
        return 0
    tiles = (s.rows // (128 // (heads // s.kv)) + len(s.spans)) * s.kv * (2 if s.hd > 256 else 1)
    assert got[0][1] % tiles == 0 and len(got) == (2 if got[0][1] > tiles else 1)
    return got[0][1] // tiles


class Filled:
    """A cache with given keys and values of every sequence up to its end, and its definition."""

    def __init__(self, g4, s, grow=0.0, positive=False, seed=0):
        self.g4, self.s = g4, s
        rng = np.random.default_rng(seed)
        ends = [p + q for p, q in s.spans]
        hist = Setup.__new__(Setup)
        hist.__dict__.update(s.__dict__)
        hist.spans, hist.offsets = [(0, e) for e in ends], np.cumsum([0] + ends).astype(np.int32)
        hist.rows = int(hist.offsets[-1])
        hist.upload()
        k, v = (tensors(rng, hist.rows, s.kv, s.hd, torch.float32) for _ in range(2))
        pos = dev(np.concatenate([np.arange(e) for e in ends]), torch.float32)
        k *= (1 + grow * pos)[:, None, None]
        if positive:
            v.abs_()
        hist.write(k, v, 0)
        self.keys, self.values = [], []
        ks, vs = ref.stored(as64(k)), ref.stored(as64(v))
        for b, e in enumerate(ends):
            at = slice(int(hist.offsets[b]), int(hist.offsets[b]) + e)
            kk, vv = ks[at].copy(), vs[at].copy()
            for p in range(0, e, s.page):
                if s.slot(b, p) is None:
                    kk[p:p + s.page] = np.nan
            self.keys.append(kk)
            self.values.append(vv)
        self.rng = rng

    def check(self, heads, name, scale, window, sample):
        s, dtype = self.s, TYPES[name]
        q = tensors(self.rng, s.rows, heads, s.hd, dtype)
        out = torch.full_like(q, 5)
        s.attend(q, out, kind_of(self.g4, name), scale, window)
        q64, got = as64(q), as64(out)
        rows = s.where()
        picked = {0, len(rows) - 1} | set(self.rng.choice(len(rows), min(sample, len(rows)), replace=False).tolist())
        for row, b, pos in (rows[i] for i in sorted(picked)):
            want, mag, delta, n = ref.attention(q64[row], self.keys[b], self.values[b], pos, scale, window)
            tol = ref.tolerance(want, mag, delta, n, torch.finfo(dtype).eps)
            err = np.abs(got[row] - want)
            assert (err <= tol).all(), (row, b, pos, float((err / tol).max()))
            if n == 0:
                assert not got[row].any()


@pytest.mark.parametrize("hd,kv,heads,page", [(64, 1, 16, 64), (128, 2, 16, 16), (256, 1, 8, 64), (512, 1, 8, 128)])
@pytest.mark.parametrize("grow,positive", [(0.0, True), (0.004, False)])
def test_sums_of_many_tiles(g4, grow, positive, hd, kv, heads, page):
    """One or two key ranges of 41 tiles: the output is summed up once to three times; values of one
    sign, and scores that rise all the way, so that the reference moves between the sums."""
    s = Setup(g4, [(0, 2600)], kv, hd, page)
    assert 41 // ranges_of(g4, s, heads, "f32") > 16
    f = Filled(g4, s, grow, positive, seed=hd)
    f.check(heads, "f32", 1 / np.sqrt(hd), 0, 24)
    f.check(heads, "f32", 1 / np.sqrt(hd), 1500, 24)


@pytest.mark.parametrize("hd", [256, 512])
def test_sums_of_runs_that_see_nothing(g4, hd):
    """The first 1100 positions have no page, and some behind them: the first sums hold nothing."""
    page = 64
    s = Setup(g4, [(0, 2500), (0, 100)], 1, hd, page)
    s.table[0, :1100 // page] = -1
    s.table[0, 30:32] = s.pages
    s.upload()
    assert 40 // ranges_of(g4, s, 8, "f32") > 16
    Filled(g4, s, 0.001, seed=hd).check(8, "f32", 1 / np.sqrt(hd), 0, 40)


@pytest.mark.parametrize("grow", [0.0, 0.002])
@pytest.mark.parametrize("hd", [256, 512])
def test_sums_in_several_ranges(g4, hd, grow):
    """Key ranges of more than 16 tiles that are joined."""
    s = Setup(g4, [(9000, 512)], 1, hd, 64)
    n = ranges_of(g4, s, 8, "f32")
    assert n > 1 and 9512 // 64 // n > 17
    Filled(g4, s, grow, grow == 0, seed=hd).check(8, "f32", 1 / np.sqrt(hd), 0, 16)


@pytest.mark.parametrize("hd,name,grow", [(64, "bf16", 0.0), (64, "f16", 0.0005), (64, "f16", 0.0),
                                          (64, "bf16", 0.0005), (512, "bf16", 0.0005)])
def test_sums_of_16_bit_types(g4, hd, name, grow):
    """More than 256 tiles in one range."""
    s = Setup(g4, [(17000, 1200 if hd == 64 else 600)], 1, hd, 128)
    assert ranges_of(g4, s, 64, name) == 1
    Filled(g4, s, grow, grow == 0, seed=hd).check(64, name, 1 / np.sqrt(hd), 0, 3)


@pytest.mark.parametrize("hd,tokens", [(64, 14), (128, 14), (256, 72), (512, 72)])
def test_either_side_of_the_bound(g4, hd, tokens):
    """The fewest rows that go to the large tiles and the most that do not, over a long context
    and a short one, with windows and softmax scales of every kind."""
    for more in (-1, 0, 3):
        s = Setup(g4, [(3000, tokens + more)], 1, hd, 64)
        assert (ranges_of(g4, s, 8, "f32") > 0) == (more >= 0)
        if more >= 0:
            assert ranges_of(g4, s, 8, "f32") > 1
        rng = np.random.default_rng(hd + more)
        check_attention(g4, s, 8, "f32", 2 / np.sqrt(hd), 0, rng)
        check_attention(g4, Setup(g4, [(3000, tokens + more)], 1, hd, 64), 8, "bf16", 2 / np.sqrt(hd), 1100, rng)
        for scale in (0.0, -0.1, 1e-30):
            check_attention(g4, Setup(g4, [(40, tokens + more)], 1, hd, 32), 8, "f32", scale, 30, rng)


@pytest.mark.parametrize("bits", [0x7F80, 0xFF80, 0x7F7F, 0xFF7F, 0xFFC0, 0x8001])
def test_unwritten_scales_behind_large_tiles(g4, bits):
    """Behind the last token scales of infinity, of the largest values, negative ones: never seen."""
    for hd in (64, 256, 512):
        fill = np.tile(np.array([bits], np.uint16).view(np.uint8), 17 * hd // 2)
        s = Setup(g4, [(40, 75)], 1, hd, 64, fill=fill)
        assert ranges_of(g4, s, 8, "f32") > 0
        check_attention(g4, s, 8, "f32", 0.1, 0, np.random.default_rng(6))


@pytest.mark.parametrize("hd,span", [(512, (131000, 1)), (256, (131000, 2)), (512, (16000, 384)), (256, (16000, 300))])
def test_error_of_fp32_outputs(g4, hd, span):
    """fp32 outputs over long contexts are within 2^-18 of 64 bits in the 2-norm (random keys and
    queries: errors of single keys are independent, so they add in squares). Few rows: p vs as two
    bf16 terms is off by up to 2^-18, evenly spread: 2^-18 / sqrt(3) = 2.2e-6. A group's score is
    four tensor-core steps that truncate by up to 2^-23 of 8 |sum q| = 64 (q of size 1): 64 2^-23
    sqrt(4 / 12), times a scale of 0.37, sqrt(8) groups and 2 / sqrt(512): 4e-7. Up to 14 steps of an
    output, each up to 2^-23 of it and always towards 0: 14 2^-24 = 8e-7. In squares 2.4e-6. Many rows:
    128 steps of an output between two sums, each of which cuts off half of 2^-24 to 2^-23 (on the
    average 0.375 2^-23) of a sum of random values, which grows like a root (2/3 on the average): 128
    2/3 0.375 2^-23 = 3.8e-6 = 2^-18. Beside it the 16 steps of the high halves of q, which shrink a
    score of size 2 by 16 / 4 2^-23 of itself (1e-6), hardly count in squares."""
    start, rows = span
    heads, n, scale = 8, start + rows, 2 / np.sqrt(hd)
    s = Setup(g4, [(0, n)], 1, hd, 64, fill=0)
    g = torch.Generator(device="cuda:0").manual_seed(hd + rows)
    k, v = (torch.randn((n, 1, hd), generator=g, device="cuda:0") for _ in range(2))
    s.write(k, v, 0)
    s.read(k, v, 0)                                     # codes times scales: exact in fp32
    s.spans, s.offsets, s.rows = [span], np.array([0, rows], np.int32), rows
    s.upload()
    q = torch.randn((rows, heads, hd), generator=g, device="cuda:0")
    out = torch.empty_like(q)
    s.attend(q, out, 0, scale, 0)
    hidden = torch.arange(n, device="cuda:0") > torch.arange(start, n, device="cuda:0")[:, None]

    exact = torch.empty(q.shape, dtype=torch.float64, device="cuda:0")
    for h in range(heads):
        sc = (q[:, h].double() @ k[:, 0].double().T * scale).masked_fill(hidden, float("-inf"))
        exact[:, h] = torch.softmax(sc, -1) @ v[:, 0].double()
    assert float((out.double() - exact).norm() / exact.norm()) <= 2.0 ** -18
