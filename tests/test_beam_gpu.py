"""Beam search's selection on the GPU against its definition in 64 bits
(tests/kv4_ref.py), and a whole search over the 4-bit cache.

Parents and tokens have to be equal. The kernel sums a row's exponentials in
fp32 per thread and joins the threads in fp64, so candidates of one beam keep
their order exactly, and candidates of two beams swap only if they are closer
than 2^-20; the seeded inputs keep them further apart or make them equal
exactly. Scores are rounded to fp32 once: half a step (2^-24 relative) and the
sum's 2^-20."""
import numpy as np
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def run(g4, x, scores, finished=None, eos=-1, ended=True, stream=None, ws=None):
    groups, beams = scores.shape
    vocab = x.shape[1]
    kind = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[x.dtype]
    d_s = torch.from_numpy(scores.astype(np.float32)).cuda()
    d_f = None if finished is None else torch.from_numpy(finished.astype(np.uint8)).cuda()
    out_s = torch.empty((groups, beams), dtype=torch.float32, device="cuda:0")
    pa, to = (torch.empty((groups, beams), dtype=torch.int32, device="cuda:0") for _ in range(2))
    fo = torch.empty((groups, beams), dtype=torch.uint8, device="cuda:0") if ended else None
    n = g4.beam_workspace(groups, beams, vocab)
    if ws is None:
        ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda:0")
    g4.beam_select(groups, beams, vocab, kind, x.data_ptr(), x.stride(0), d_s.data_ptr(),
                   None if d_f is None else d_f.data_ptr(), eos, out_s.data_ptr(), pa.data_ptr(), to.data_ptr(),
                   fo.data_ptr() if ended else None, ws.data_ptr(), ws.numel(), stream)
    torch.cuda.synchronize()
    return [None if t is None else t.cpu().numpy() for t in (out_s, pa, to, fo)]


def check(g4, x, scores, finished=None, eos=-1):
    groups, beams = scores.shape
    got = run(g4, x, scores, finished, eos)
    x64 = x.double().cpu().numpy().reshape(groups, beams, -1)
    for g in range(groups):
        fin = None if finished is None else finished[g]
        s, pa, to, en = ref.beam(x64[g], scores[g].astype(np.float32).astype(np.float64), fin, eos)
        assert got[1][g].tolist() == pa.tolist() and got[2][g].tolist() == to.tolist(), (g, got[1][g], pa)
        assert got[3][g].astype(bool).tolist() == en.tolist()
        inf = ~np.isfinite(s)
        assert np.array_equal(got[0][g][inf], s[inf].astype(np.float32))
        assert (np.abs(got[0][g][~inf] - s[~inf]) <= 2.0 ** -24 * np.abs(s[~inf]) + 2.0 ** -20).all()
    return got


def inputs(rng, groups, beams, vocab, dtype, pad=0):
    x = torch.from_numpy((4 * rng.standard_normal((groups * beams, vocab + pad))).astype(np.float32)).to(dtype).cuda()
    return x[:, :vocab], -20 * rng.random((groups, beams))


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("groups,beams,vocab,pad", [(1, 1, 1, 0), (1, 4, 3, 0), (2, 8, 8, 0), (3, 5, 1000, 24),
                                                    (1, 32, 4097, 0), (2, 3, 8193, 7), (1, 4, 50001, 0),
                                                    (1, 4, 262144, 0)])
def test_select(g4, name, groups, beams, vocab, pad):
    rng = np.random.default_rng(vocab + beams)
    x, scores = inputs(rng, groups, beams, vocab, TYPES[name], pad)
    check(g4, x, scores)
    if vocab > 2:
        fin = rng.random((groups, beams)) < 0.4
        check(g4, x, scores, fin, eos=2)
        check(g4, x, scores, fin, eos=vocab - 1)
        check(g4, x, scores, np.ones_like(fin), eos=1)


def test_ties_go_to_the_lowest_index(g4):
    """Equal logits in a row, equal rows, whole rows of one value (more ties than any buffer)."""
    for vocab, dtype in ((20000, torch.float32), (9000, torch.bfloat16), (300, torch.float16)):
        x = torch.zeros((4, vocab), dtype=dtype, device="cuda:0")
        check(g4, x, np.zeros((1, 4)))
        check(g4, x, np.array([[-1.0, 0.0, 0.0, -2.0]]))
        x[:, vocab // 2] = 3
        x[:, vocab // 2 + 5] = 3
        x[:, 7] = 3
        check(g4, x, np.zeros((1, 4)))
        x[2, 11] = 3
    x = torch.zeros((2, 64), dtype=torch.float32, device="cuda:0")
    x[0, 40], x[0, 3] = 0.0, -0.0                      # one value
    check(g4, x, np.zeros((1, 2)))


def test_masked_and_special_values(g4):
    rng = np.random.default_rng(4)
    inf = float("inf")
    x, scores = inputs(rng, 1, 4, 5000, torch.float32)
    x = x.clone()
    x[0, 10:] = -inf                                   # few tokens left
    x[1] = -inf                                        # none left
    x[2, ::3] = float("nan")
    x[3, 5:] = torch.finfo(torch.float32).min
    check(g4, x, scores)
    check(g4, x, np.array([[-inf, -1.0, -inf, -inf]]))  # first step: one live beam, and that one without tokens
    check(g4, x, np.array([[0.0, -inf, -inf, -inf]]))
    check(g4, x, np.full((1, 4), -inf))
    check(g4, x, np.array([[float("nan"), inf, -3.0, -2.0]]), np.array([[True, True, False, True]]), eos=4000)
    x[0, 3] = inf                                      # no softmax: the row's candidates are not numbers
    check(g4, x, scores)
    x[:] = -inf
    check(g4, x, scores)
    check(g4, x, scores, np.array([[False, True, False, True]]), eos=3)


def best(row, count):
    """The `count` best tokens of a row and their log softmax in 64 bits, the maximum taken off
    first: beside one of 1e10 the logarithm of the sum would be lost."""
    x = row.double().cpu().numpy()
    x = np.where(np.isnan(x), -np.inf, x)
    d = x - x.max()
    at = np.lexsort((np.arange(len(x)), -x))[:count]
    return at, d[at] - np.log(np.exp(d).sum())


def alone(g4, row):
    """A row that has to win: as a search of its own, with one beam and with beams far behind it."""
    vocab = row.shape[-1]
    got = run(g4, row.reshape(1, vocab).contiguous(), np.array([[-1.5]]))
    at, s = best(row, 1)
    assert got[2].tolist() == [at.tolist()]
    assert abs(got[0][0, 0] - (s[0] - 1.5)) <= 2.0 ** -24 * abs(s[0] - 1.5) + 2.0 ** -20
    x = torch.zeros((4, vocab), dtype=row.dtype, device="cuda:0")
    x[2] = row
    got = run(g4, x, np.array([[-5000.0, -5000.0, 0.0, -5000.0]]))
    at, s = best(row, 4)
    n = int((s > -4000).sum())                          # the others come from the beams behind
    assert n >= 1 and got[1][0, :n].tolist() == [2] * n and got[2][0, :n].tolist() == at[:n].tolist()
    assert (got[1][0, n:] != 2).all()
    assert (np.abs(got[0][0, :n] - s[:n]) <= 2.0 ** -24 * np.abs(s[:n]) + 2.0 ** -20).all()


FAR = {"f32": (-3.4028234663852886e38, -1e30, -1e10, -3e9, -2.0 ** 28 - 32, -2.0 ** 28, 2.0 ** 28 + 32, 1e10, 3e38),
       "bf16": (-3.3895313892515355e38, -1e30, -1e10, -3e9, 2.0 ** 28 + 2.0 ** 21, 3e38), "f16": (-65504.0, 65504.0)}


@pytest.mark.parametrize("name,value", [(n, v) for n, vs in FAR.items() for v in vs])
@pytest.mark.parametrize("vocab", [7, 5000, 70001])
def test_far_logits(g4, name, value, vocab):
    """Finite logits of any size (a vocabulary masked with the type's lowest value or -1e10):
    rows of them alone, with one token left, with parts of the row left, and neighbouring values
    that are still within a few units of each other. Each row is checked where it wins."""
    dtype = TYPES[name]
    rng = np.random.default_rng(vocab)
    far = torch.full((vocab,), value, dtype=dtype, device="cuda:0")
    live = torch.from_numpy(rng.standard_normal(vocab).astype(np.float32)).to(dtype).cuda()
    alone(g4, far)
    for keep in (slice(vocab // 2, vocab // 2 + 1), slice(0, vocab // 2), slice(vocab // 2, None)):
        x = far.clone()
        x[keep] = live[keep]
        alone(g4, x)
    x = far.clone()
    x[::3] = torch.nextafter(far[0], torch.zeros_like(far[0]))
    x[1::3] = torch.nextafter(x[0], torch.zeros_like(far[0]))
    alone(g4, x)
    x[vocab // 2] = float("nan")                        # summed up once more without it
    alone(g4, x)
    x = far.clone()
    x[vocab // 3:] = float("-inf")
    alone(g4, x)


def test_far_logits_rise_and_fall(g4):
    """Sizes that change from chunk to chunk of a slice: the running maximum crosses every form of the sum."""
    steps = [-3.4028234663852886e38, -1e30, -1e10, -2.0 ** 28 - 32, -2.0 ** 28, -1e6, -3.0, 2.0, 1e6, 2.0 ** 28,
             2.0 ** 28 + 32, 1e10, 3e38]
    # 64 searches of 4 beams leave one slice of several chunks per row
    for order in (steps, steps[::-1], steps[::2] + steps[1::2]):
        row = torch.tensor(np.repeat(np.array(order, np.float32), 4096), device="cuda:0")
        for last in range(1, len(order) + 1):
            x = torch.zeros((4 * 64, last * 4096), device="cuda:0")
            x[2::4] = row[:last * 4096]
            got = run(g4, x, np.tile(np.array([[-5000.0, -5000.0, 0.0, -5000.0]]), (64, 1)))
            top = row[:last * 4096].double()
            want = -np.log(float((top - top.max()).exp().sum()))
            assert (got[1][:, 0] == 2).all() and (got[2][:, 0] == int(top.argmax())).all(), (order, last)
            assert (np.abs(got[0][:, 0] - want) <= 2.0 ** -24 * abs(want) + 2.0 ** -20).all(), (order, last)


def test_special_rows_win(g4):
    """Every kind of special row as the row that wins: few tokens left, NaN among them, one value."""
    rng = np.random.default_rng(8)
    inf, nan = float("inf"), float("nan")
    x = torch.from_numpy(rng.standard_normal(5000).astype(np.float32)).cuda()
    for change in (lambda r: r[10:].fill_(-inf), lambda r: r[:4990].fill_(-inf), lambda r: r[::3].fill_(nan),
                   lambda r: r[5:].fill_(torch.finfo(torch.float32).min), lambda r: r[1:].fill_(nan)):
        row = x.clone()
        change(row)
        for dtype in TYPES.values():
            alone(g4, row.clamp(min=torch.finfo(dtype).min).where(row != -inf, row).to(dtype))


def test_peaked_rows(g4):
    """One token holds nearly all probability; the others' order survives."""
    x = torch.full((2, 100000), -30.0, device="cuda:0")
    x[0, 77], x[1, 99999] = 60.0, 55.0
    x[0, 5], x[1, 6], x[0, 3] = 20.0, 19.0, 18.5
    check(g4, x, np.array([[-1.0, -1.25]]))


def test_offsets_beyond_32_bits(g4):
    """A row stride that puts the last row beyond 2^32 bytes."""
    vocab, stride = 3000, (1 << 30) + 16
    x = torch.empty(stride + vocab, dtype=torch.float32, device="cuda:0").as_strided((2, vocab), (stride, 1))
    rng = np.random.default_rng(1)
    x.copy_(torch.from_numpy(rng.standard_normal((2, vocab)).astype(np.float32)))
    check(g4, x, np.array([[-1.0, -0.5]]))


def test_no_finished_output_and_streams(g4):
    rng = np.random.default_rng(6)
    x, scores = inputs(rng, 2, 4, 30000, torch.float32)
    want = run(g4, x, scores, eos=9)
    got = run(g4, x, scores, eos=9, ended=False)
    assert got[3] is None and all(np.array_equal(a, b) for a, b in zip(got[:3], want[:3]))
    # another alignment of the same logits: the same selection and scores
    y = torch.empty((8, 30003), dtype=torch.float32, device="cuda:0")[:, 1:30001]
    y.copy_(x)
    assert all(np.array_equal(a, b) for a, b in zip(run(g4, y, scores, eos=9), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(np.array_equal(a, b) for a, b in zip(run(g4, x, scores, eos=9, stream=side.cuda_stream), want))


def test_search_over_the_cache(g4):
    """Beams decoded over shared pages: write, attend, select, reorder, for
    enough steps to fill pages, captured into one graph per parity of the
    ping-pong tables; against a search that keeps every beam's values apart."""
    groups, beams, kv, hd, heads, page, vocab, steps = 2, 3, 1, 64, 4, 16, 500, 40
    prompt = [21, 5]
    rng = np.random.default_rng(12)
    rows = groups * beams
    emb = rng.standard_normal((vocab, (heads + 2 * kv) * hd)).astype(np.float32)
    head = (rng.standard_normal((heads * hd, vocab)) * 0.4).astype(np.float32)
    d_emb, d_head = torch.from_numpy(emb).cuda(), torch.from_numpy(head).double().cuda()
    most = max(prompt) + steps
    stride = most // page + 2
    pages = rows * (stride + 1)
    pool = torch.full((pages * g4.kv4_page_bytes(kv, hd, page),), 0xFF, dtype=torch.uint8, device="cuda:0")
    ids = rng.permutation(pages).astype(np.int32)
    table = ids[:rows * stride].reshape(rows, stride).copy()
    for g in range(groups):                    # the prompt's full pages are shared
        full = prompt[g] // page
        table[g * beams:(g + 1) * beams, :full] = table[g * beams, :full]
    tables = [torch.from_numpy(table).cuda(), torch.empty((rows, stride), dtype=torch.int32, device="cuda:0")]
    spares = [torch.from_numpy(ids[rows * stride:]).cuda(), torch.empty(rows, dtype=torch.int32, device="cuda:0")]
    cache = g4.Kv4Cache(pool.data_ptr(), pages, page, kv, hd)
    caches = g4.kv4_caches([cache])

    # prompts: every beam writes its own copy of the tokens (the shared pages get the same ones)
    toks = [rng.integers(0, vocab, p) for p in prompt]
    all_rows = np.concatenate([np.tile(toks[g], beams) for g in range(groups)])
    x = d_emb[torch.from_numpy(all_rows).cuda()].contiguous()
    counts = [p for p in prompt for _ in range(beams)]
    for g in range(groups):                    # one beam at a time: no two rows of a call name a slot
        for w in range(beams):
            i = g * beams + w
            at = sum(counts[:i])
            off, st = torch.tensor([0, prompt[g]], dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
            b = g4.Kv4Batch(1, prompt[g], off.data_ptr(), st.data_ptr(), tables[0][i].data_ptr(), stride)
            k = x[at:at + prompt[g], heads * hd:]
            g4.kv4_write(cache, b, 0, k.data_ptr(), x.stride(0), k.data_ptr() + kv * hd * 4, x.stride(0))
            torch.cuda.synchronize()
    # the definition's side: every beam's stored keys and values
    hist = [[list(map(lambda t: ref.stored(emb[t].astype(np.float64)[heads * hd:].reshape(2, hd)), toks[g]))
             for _ in range(beams)] for g in range(groups)]
    tokens = np.array([[toks[g][-1]] * beams for g in range(groups)])
    scores = np.array([[0.0] + [-np.inf] * (beams - 1)] * groups)
    finished = np.zeros((groups, beams), bool)
    eos = 3

    lengths = torch.tensor(prompt, dtype=torch.int32).cuda()
    start = lengths.repeat_interleave(beams).contiguous()
    offsets = torch.arange(rows + 1, dtype=torch.int32).cuda()
    d_tok = torch.from_numpy(tokens.ravel().astype(np.int32)).cuda()
    d_sc = [torch.from_numpy(scores.astype(np.float32)).cuda(), torch.empty((groups, beams), device="cuda:0")]
    d_fin = [torch.zeros((groups, beams), dtype=torch.uint8, device="cuda:0") for _ in range(2)]
    parents = torch.empty((groups, beams), dtype=torch.int32, device="cuda:0")
    out = torch.empty((rows, heads, hd), device="cuda:0")
    logits = torch.empty((rows, vocab), device="cuda:0")
    row = torch.empty((rows, (heads + 2 * kv) * hd), device="cuda:0")
    batches = [g4.Kv4Batch(rows, rows, offsets.data_ptr(), start.data_ptr(), t.data_ptr(), stride) for t in tables]
    ws = torch.empty(max(g4.kv4_attention_workspace(cache, batches[0], 0, heads),
                         g4.beam_workspace(groups, beams, vocab)), dtype=torch.uint8, device="cuda:0")

    def step(i, st):
        a, b = i % 2, 1 - i % 2
        torch.index_select(d_emb, 0, d_tok, out=row)
        k = row.data_ptr() + heads * hd * 4
        g4.kv4_write(cache, batches[a], 0, k, row.stride(0), k + kv * hd * 4, row.stride(0), st)
        g4.kv4_attention(cache, batches[a], 0, heads, row.data_ptr(), row.stride(0), out.data_ptr(), heads * hd, 0.125,
                         0, ws.data_ptr(), ws.numel(), st)
        logits.copy_(out.reshape(rows, -1).double() @ d_head)
        g4.beam_select(groups, beams, vocab, 0, logits.data_ptr(), vocab, d_sc[a].data_ptr(), d_fin[a].data_ptr(), eos,
                       d_sc[b].data_ptr(), parents.data_ptr(), d_tok.data_ptr(), d_fin[b].data_ptr(), ws.data_ptr(),
                       ws.numel(), st)
        lengths.add_(1)
        start.add_(1)
        g4.kv4_reorder(caches, groups, beams, parents.data_ptr(), lengths.data_ptr(), tables[a].data_ptr(),
                       tables[b].data_ptr(), stride, spares[a].data_ptr(), spares[b].data_ptr(), st)

    step(0, torch.cuda.current_stream().cuda_stream)
    graphs = []
    for i in (1, 0):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            step(i, torch.cuda.current_stream().cuda_stream)
        graphs.append(gr)
    moved = 0
    for i in range(steps):
        if i:
            graphs[(i - 1) % 2].replay()
        torch.cuda.synchronize()
        x64 = emb.astype(np.float64)
        lg = np.zeros((groups, beams, vocab))
        for g in range(groups):
            for w in range(beams):
                t = tokens[g, w]
                hist[g][w] = hist[g][w] + [ref.stored(x64[t][heads * hd:].reshape(2, hd))]
                kvs = np.stack(hist[g][w])
                o, *_ = ref.attention(x64[t][:heads * hd].reshape(heads, hd), kvs[:, :1], kvs[:, 1:], len(kvs) - 1,
                                      0.125, 0)
                lg[g, w] = o.ravel() @ head.astype(np.float64)
        got_p, got_t = parents.cpu().numpy(), d_tok.cpu().numpy().reshape(groups, beams)
        got_s = d_sc[1 - i % 2].cpu().numpy()
        for g in range(groups):
            s, pa, to, en = ref.beam(lg[g], scores[g], finished[g], eos)
            assert got_p[g].tolist() == pa.tolist() and got_t[g].tolist() == to.tolist(), (i, g)
            assert np.abs(got_s[g] - s).max() < 1e-3 * (i + 1)
            moved += int((pa != np.arange(beams)).sum())
            hist[g] = [list(hist[g][p]) for p in pa]
            scores[g], tokens[g], finished[g] = s, to, en
    assert moved > 10
    # what the caches hold at the end is what every beam's history says
    a = steps % 2
    for g in range(groups):
        n = prompt[g] + steps
        for w in range(beams):
            off, st = torch.tensor([0, n], dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
            b = g4.Kv4Batch(1, n, off.data_ptr(), st.data_ptr(), tables[a][g * beams + w].data_ptr(), stride)
            ko, vo = torch.empty((n, hd), device="cuda:0"), torch.empty((n, hd), device="cuda:0")
            g4.kv4_read(cache, b, 0, ko.data_ptr(), hd, vo.data_ptr(), hd)
            kvs = np.stack(hist[g][w])
            assert np.array_equal(ko.cpu().numpy(), kvs[:, 0].astype(np.float32))
            assert np.array_equal(vo.cpu().numpy(), kvs[:, 1].astype(np.float32))
