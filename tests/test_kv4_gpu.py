"""The paged 4-bit KV cache on the GPU: quantising writes, reads, attention and
the reordering of a beam search's caches, each against its definition in 64
bits (tests/kv4_ref.py). Writes, reads and reorderings are compared byte for
byte, attention within the bound that kv4_ref.tolerance derives."""
import numpy as np
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def dev(x, dtype=torch.int32):
    return torch.as_tensor(np.asarray(x)).to(dtype).to("cuda:0")


def as64(t):
    return t.detach().to("cpu", torch.float64).numpy()


class Setup:
    """A pool on the GPU with its copy on the CPU, and a batch of rows."""

    def __init__(self, g4, spans, kv, hd, page, fill=0xFF, rows=None, spare_pages=3, stride=None, seed=0):
        self.g4, self.kv, self.hd, self.page = g4, kv, hd, page
        rng = np.random.default_rng(seed)
        held = [max(0, -(-(p + q) // page)) for p, q in spans]
        total = sum(held) + spare_pages
        ids = rng.permutation(total).astype(np.int32)
        self.table = np.full((len(spans), stride or max(held + [1])), -1, np.int32)
        at = 0
        for i, m in enumerate(held):
            self.table[i, :m] = ids[at:at + m]
            at += m
        self.spans, self.pages = spans, total
        self.offsets = np.cumsum([0] + [q for _, q in spans]).astype(np.int32)
        self.rows = int(self.offsets[-1]) if rows is None else rows
        self.ref = ref.Cache(total, page, kv, hd, fill)
        self.pool = dev(self.ref.bytes, torch.uint8)
        self.upload()

    def upload(self):
        self.d_off, self.d_start = dev(self.offsets), dev([p for p, _ in self.spans])
        self.d_table = dev(self.table)
        self.cache = self.g4.Kv4Cache(self.pool.data_ptr(), self.pages, self.page, self.kv, self.hd)
        self.batch = self.g4.Kv4Batch(len(self.spans), self.rows, self.d_off.data_ptr(), self.d_start.data_ptr(),
                                      self.d_table.data_ptr(), self.table.shape[1])

    def where(self):
        """(row, sequence, position) of every row that belongs to one."""
        return [(int(self.offsets[b]) + i, b, p + i) for b, (p, q) in enumerate(self.spans) for i in range(q)]

    def slot(self, b, pos):
        j = pos // self.page
        if pos < 0 or j >= self.table.shape[1] or not 0 <= self.table[b, j] < self.pages:
            return None
        return int(self.table[b, j]), pos % self.page

    def write(self, k, v, kind, stream=None):
        self.g4.kv4_write(self.cache, self.batch, kind, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), stream)

    def read(self, k, v, kind, stream=None):
        self.g4.kv4_read(self.cache, self.batch, kind, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), stream)

    def attend(self, q, out, kind, scale, window, ws=None, stream=None):
        n = self.g4.kv4_attention_workspace(self.cache, self.batch, kind, q.shape[1])
        if ws is None:
            ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda:0")
        assert ws.numel() >= n
        self.g4.kv4_attention(self.cache, self.batch, kind, q.shape[1], q.data_ptr(), q.stride(0), out.data_ptr(),
                              out.stride(0), scale, window, ws.data_ptr(), ws.numel(), stream)
        return ws


def kind_of(g4, name):
    return getattr(g4, "TYPE_" + name.upper())


def tensors(rng, rows, heads, hd, dtype, pad=0):
    """Rows of `heads` heads inside wider rows (pad more elements)."""
    x = torch.from_numpy(rng.standard_normal((max(rows, 1), heads * hd + pad)).astype(np.float32)).to(dtype).to("cuda:0")
    return x.as_strided((rows, heads, hd), (heads * hd + pad, hd, 1))


# spans: one token; a chunk inside a page; across pages; padding; empty sequences; many
SPANS = {
    "one": [(0, 1)],
    "inside": [(5, 7)],
    "across": [(13, 55)],
    "ragged": [(0, 3), (31, 1), (7, 0), (16, 16), (100, 29)],
    "padded": [(-5, 9), (-40, 8), (-16, 17)],
    "step": [(p, 1) for p in (0, 15, 16, 63, 64, 200)],
}


@pytest.mark.parametrize("hd,kv,page", [(64, 1, 16), (128, 3, 32), (256, 1, 64), (512, 2, 128)])
@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("spans", list(SPANS))
def test_write_and_read(g4, spans, name, hd, kv, page):
    rng = np.random.default_rng(len(spans) + len(name) + hd)
    s = Setup(g4, SPANS[spans], kv, hd, page)
    dtype = TYPES[name]
    k, v = (tensors(rng, s.rows, kv, hd, dtype, pad) for pad in (0, 64))
    k64, v64 = as64(k), as64(v)
    s.write(k, v, kind_of(g4, name))
    ko, vo = torch.full_like(k, 7), torch.full_like(v, 7)
    s.read(ko, vo, kind_of(g4, name))
    torch.cuda.synchronize()
    want = [torch.zeros_like(ko), torch.zeros_like(vo)]
    for row, b, pos in s.where():
        at = s.slot(b, pos)
        if at:
            for h in range(kv):
                s.ref.put(at[0], at[1], h, k64[row, h], v64[row, h])
            for w, x in zip(want, (k64, v64)):
                w[row] = torch.from_numpy(ref.stored(x[row])).to(dtype)
    assert np.array_equal(s.pool.cpu().numpy(), s.ref.bytes)      # nothing else of the pool is touched
    for got, w in zip((ko, vo), want):
        assert torch.equal(got.float(), w.float())


def test_write_special_groups(g4):
    """Non-finite values, groups of zeros and of tiny values, ties, the largest finite values."""
    s = Setup(g4, [(3, 8)], 1, 64, 16)
    x = np.zeros((8, 1, 64), np.float32)
    x[0, 0, :6] = [7, 0.5, 1.5, 2.5, -0.5, -3.5]
    x[1, 0, 5] = np.nan
    x[2, 0, 5] = -np.inf
    x[3, 0, 9] = 2.0 ** -101
    x[4, 0] = np.linspace(-1, 1, 64) * 3e-38
    x[5, 0] = np.linspace(-1, 1, 64) * np.float32(1.6e38)
    x[6, 0, :4] = [7, np.nextafter(np.float32(0.5), np.float32(0)), np.nextafter(np.float32(2.5), np.float32(9)), -7]
    x[7, 0] = -0.0
    k = dev(x, torch.float32)
    ko, vo = torch.empty_like(k), torch.empty_like(k)
    s.write(k, k, 0)
    s.read(ko, vo, 0)
    want = ref.stored(x.astype(np.float64)).astype(np.float32)
    for got in (ko, vo):
        got = got.cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert np.array_equal(np.nan_to_num(got), np.nan_to_num(want))


def test_codes_next_to_borders(g4):
    """Values one fp32 step either side of every border between two codes."""
    s = Setup(g4, [(0, 64)], 1, 64, 64)
    rng = np.random.default_rng(3)
    x = np.zeros((64, 1, 64), np.float32)
    for i in range(64):
        sc = float(ref.bf16(np.float64(rng.uniform(1e-3, 10))))
        x[i, 0, 0] = 7 * sc
        b = np.float32((np.arange(-7, 7) + 0.5) * sc)
        x[i, 0, 1:15] = b
        x[i, 0, 15:29] = np.nextafter(b, np.float32(-1e9))
        x[i, 0, 29:43] = np.nextafter(b, np.float32(1e9))
    k = dev(x, torch.float32)
    ko, vo = torch.empty_like(k), torch.empty_like(k)
    s.write(k, k, 0)
    s.read(ko, vo, 0)
    want = ref.stored(x.astype(np.float64)).astype(np.float32)
    assert np.array_equal(ko.cpu().numpy(), want) and np.array_equal(vo.cpu().numpy(), want)


def test_rows_without_pages(g4):
    """Bad page numbers and positions past the table: dropped, read as 0, nothing else touched."""
    s = Setup(g4, [(0, 40), (30, 20)], 2, 64, 16)
    s.table[0, 1] = s.pages            # out of range
    s.table[1, 2] = -7
    s.table[1, 3] = 2 ** 31 - 1
    s.upload()
    rng = np.random.default_rng(0)
    k, v = tensors(rng, s.rows, 2, 64, torch.float32), tensors(rng, s.rows, 2, 64, torch.float32)
    s.write(k, v, 0)
    ko, vo = torch.full_like(k, 5), torch.full_like(v, 5)
    s.read(ko, vo, 0)
    k64, v64 = as64(k), as64(v)
    for row, b, pos in s.where():
        at = s.slot(b, pos)
        if at is None:
            assert not ko[row].any() and not vo[row].any()
        else:
            for h in range(2):
                s.ref.put(at[0], at[1], h, k64[row, h], v64[row, h])
            assert np.array_equal(as64(ko[row]), ref.stored(k64[row]).astype(np.float32))
    assert np.array_equal(s.pool.cpu().numpy(), s.ref.bytes)
    short = Setup(g4, [(0, 40)], 1, 64, 16, stride=3)
    short.batch.table_stride = 2       # positions 32..39 are past the table
    k = tensors(rng, 40, 1, 64, torch.float32)
    short.write(k, k, 0)
    ko, vo = torch.full_like(k, 5), torch.full_like(k, 5)
    short.read(ko, vo, 0)
    assert not ko[32:].any() and ko[:32].any(-1).all()


def test_rows_behind_the_last_sequence(g4):
    s = Setup(g4, [(4, 3), (0, 5)], 1, 128, 16, rows=20)
    rng = np.random.default_rng(1)
    k, v = tensors(rng, 20, 1, 128, torch.bfloat16), tensors(rng, 20, 1, 128, torch.bfloat16)
    s.write(k, v, 1)
    ko, vo = torch.full_like(k, 5), torch.full_like(v, 5)
    s.read(ko, vo, 1)
    q = tensors(rng, 20, 4, 128, torch.bfloat16)
    out = torch.full_like(q, 5)
    s.attend(q, out, 1, 0.1, 0)
    torch.cuda.synchronize()
    for x in (ko, vo, out):
        assert (x[8:] == 5).all() and (x[:8] != 5).any()


def check_attention(g4, s, heads, name, scale, window, rng, pad=0, q_scale=1.0):
    """Fill the cache with the rows' history, attend, compare with the definition."""
    kv, hd, dtype = s.kv, s.hd, TYPES[name]
    ends = [max(0, p + q) for p, q in s.spans]
    hist = Setup.__new__(Setup)
    hist.__dict__.update(s.__dict__)
    hist.spans = [(0, e) for e in ends]
    hist.offsets = np.cumsum([0] + ends).astype(np.int32)
    hist.rows = int(hist.offsets[-1])
    hist.upload()
    keys = [np.full((e, kv, hd), np.nan) for e in ends]
    values = [np.full((e, kv, hd), np.nan) for e in ends]
    if hist.rows:
        k, v = tensors(rng, hist.rows, kv, hd, torch.float32), tensors(rng, hist.rows, kv, hd, torch.float32)
        hist.write(k, v, 0)
        ks, vs = ref.stored(as64(k)), ref.stored(as64(v))
        for row, b, pos in hist.where():
            if hist.slot(b, pos):
                keys[b][pos], values[b][pos] = ks[row], vs[row]
    q = tensors(rng, s.rows, heads, hd, dtype, pad)
    q.mul_(q_scale)
    out = torch.full_like(q, 5)
    s.attend(q, out, kind_of(g4, name), scale, window)
    q64, got = as64(q), as64(out)
    worst = 0.0
    for row, b, pos in s.where():
        want, mag, delta, n = ref.attention(q64[row], keys[b], values[b], pos, scale, window)
        tol = ref.tolerance(want, mag, delta, n, torch.finfo(dtype).eps)
        err = np.abs(got[row] - want)
        worst = max(worst, float((err / tol).max()))
        assert (err <= tol).all(), (row, b, pos, float((err / tol).max()))
        if n == 0:
            assert not got[row].any()
    return q, out


ATTN_SPANS = {
    "first": [(0, 1)],
    "one": [(36, 1)],
    "records": [(p, 1) for p in (14, 15, 16, 31, 32, 33, 127, 128, 300)],
    "chunk": [(11, 37)],
    "prompt": [(0, 70)],
    "ragged": [(0, 3), (61, 1), (9, 0), (200, 18), (16, 16)],
    "padded": [(-5, 9), (-40, 8), (-1, 2), (20, 1)],
}


@pytest.mark.parametrize("hd,kv,heads,page", [(64, 2, 2, 16), (64, 1, 16, 64), (128, 2, 8, 32), (256, 1, 8, 64),
                                              (256, 2, 10, 16), (512, 1, 8, 64), (512, 1, 24, 128)])
@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("spans", list(ATTN_SPANS))
def test_attention(g4, spans, name, hd, kv, heads, page):
    rng = np.random.default_rng(len(spans) + hd + heads)
    s = Setup(g4, ATTN_SPANS[spans], kv, hd, page)
    check_attention(g4, s, heads, name, 1.5 / np.sqrt(hd), 0, rng)


@pytest.mark.parametrize("window", [1, 5, 16, 40, 1000])
@pytest.mark.parametrize("hd,heads", [(64, 4), (256, 8), (512, 8)])
def test_attention_window(g4, window, hd, heads):
    rng = np.random.default_rng(window)
    s = Setup(g4, [(300, 1), (0, 50), (97, 33), (-3, 5)], 1, hd, 32)
    check_attention(g4, s, heads, "f32", 0.2, window, rng, pad=128)


@pytest.mark.parametrize("hd,heads,kv", [(64, 8, 1), (128, 6, 2), (256, 8, 1), (512, 8, 1)])
@pytest.mark.parametrize("n", [1, 40, 140])
def test_attention_items_of_few_records(g4, n, hd, heads, kv):
    """Windows and tables of few records, where a CTA has an item for itself, beside ones
    that are just too long or too many for that; empty sequences and rows between them."""
    rng = np.random.default_rng(n)
    spans = [(int(p), int(rng.integers(0, 4))) for p in rng.integers(0, 900, n)]
    for window in (17, 600, 640, 1016, 1017):
        check_attention(g4, Setup(g4, spans, kv, hd, 64), heads, "f32", 0.1, window, rng)
    check_attention(g4, Setup(g4, [(p % 200, q) for p, q in spans], kv, hd, 16), heads, "bf16", 0.1, 0, rng)


@pytest.mark.parametrize("hd,heads,kv,name", [(512, 8, 1, "f32"), (256, 8, 1, "f32"), (128, 32, 8, "bf16"),
                                              (64, 8, 1, "f16")])
def test_attention_long(g4, hd, heads, kv, name):
    """Contexts that are split over CTAs and joined, peaked and flat scores."""
    rng = np.random.default_rng(hd)
    s = Setup(g4, [(5003, 1), (1, 1), (2999, 2)], kv, hd, 128)
    check_attention(g4, s, heads, name, 1 / np.sqrt(hd), 0, rng, q_scale=4.0)
    s = Setup(g4, [(9001, 1)], kv, hd, 64)
    check_attention(g4, s, heads, name, 1e-3, 0, rng)


@pytest.mark.parametrize("hd,heads,kv,name", [(512, 8, 1, "f32"), (256, 8, 1, "bf16"), (128, 16, 4, "f32"),
                                              (64, 6, 2, "f16"), (128, 64, 1, "bf16")])
def test_attention_prompts(g4, hd, heads, kv, name):
    """Long chunks: whole prompts, a chunk behind a context, mixed with single tokens."""
    rng = np.random.default_rng(heads)
    s = Setup(g4, [(0, 150), (700, 1), (333, 129), (-20, 30)], kv, hd, 64)
    check_attention(g4, s, heads, name, 1 / np.sqrt(hd), 0, rng)
    check_attention(g4, s, heads, name, 1 / np.sqrt(hd), 100, rng)


PROMPT_SPANS = {
    "whole": [(0, 150)],
    "behind": [(333, 129)],
    "mixed": [(0, 131), (700, 1), (61, 260), (-20, 90), (5, 0)],
}


@pytest.mark.parametrize("hd,kv,heads,page", [(64, 2, 8, 16), (64, 1, 64, 64), (128, 2, 10, 32), (128, 1, 3, 1024),
                                              (256, 1, 8, 64), (256, 2, 8, 128), (512, 1, 8, 64), (512, 2, 10, 16)])
@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("spans", list(PROMPT_SPANS))
def test_prompt_tiles(g4, spans, name, hd, kv, heads, page):
    """Row counts that go to the tiles of 128 rows: whole prompts, chunks inside
    pages and tiles, sequences of one token among them, padding, tiles that the
    heads of a group do not fill, windows."""
    rng = np.random.default_rng(hd + heads)
    s = Setup(g4, PROMPT_SPANS[spans], kv, hd, page)
    check_attention(g4, s, heads, name, 1 / np.sqrt(hd), 0, rng, q_scale=2.0)
    check_attention(g4, s, heads, name, -0.5 / np.sqrt(hd), 77, rng, pad=64)


@pytest.mark.parametrize("hd,heads", [(64, 8), (256, 8), (512, 8)])
def test_prompt_tiles_split(g4, hd, heads):
    """Few row tiles over a long context: key ranges joined, with rows that see only some."""
    rng = np.random.default_rng(hd)
    check_attention(g4, Setup(g4, [(3000, 70)], 1, hd, 64), heads, "f32", 2 / np.sqrt(hd), 0, rng)
    check_attention(g4, Setup(g4, [(3000, 70)], 1, hd, 64), heads, "bf16", 2 / np.sqrt(hd), 1100, rng)


def test_prompt_tiles_window_needs_no_more_workspace(g4):
    """The workspace is asked for without the window: every window fits into it."""
    s = Setup(g4, [(0, 150)], 1, 256, 16, stride=4096)
    for window in (1, 16, 64, 500, 20000, 2 ** 31 - 1):
        check_attention(g4, s, 8, "bf16", 0.1, window, np.random.default_rng(window))


@pytest.mark.parametrize("hd", [64, 512])
def test_prompt_tiles_pages_missing(g4, hd):
    """Missing pages, among them all of a row tile's, and pages past the table."""
    s = Setup(g4, [(100, 140), (20, 130), (90, 140), (0, 200)], 1, hd, 16)
    s.table[0, 2] = -1
    s.table[0, 6] = s.pages + 3
    s.table[1, :] = -1
    s.table[2, 3:9] = 2 ** 31 - 1
    s.table[3, :5] = -9
    s.upload()
    check_attention(g4, s, 8, "f32", 0.1, 0, np.random.default_rng(5))


@pytest.mark.parametrize("hd", [128, 512])
def test_prompt_tiles_nan_and_infinity(g4, hd):
    """A key or value that is not finite reaches the rows that see it (a value: the
    dimensions of its group), and no other row, though they share its tile."""
    s = Setup(g4, [(0, 200)], 1, hd, 64)
    rng = np.random.default_rng(7)
    k, v = tensors(rng, 200, 1, hd, torch.float32), tensors(rng, 200, 1, hd, torch.float32)
    v[33, 0, 70] = float("nan")
    k[150, 0, 3] = float("inf")
    s.write(k, v, 0)
    q = tensors(rng, 200, 8, hd, torch.float32)
    q[20, 3, 5] = float("inf")
    for window in (0, 60):
        out = torch.empty_like(q)
        s.attend(q, out, 0, 0.1, window)
        for row in range(200):
            bad = torch.zeros((8, hd), dtype=torch.bool, device="cuda:0")
            if 33 <= row and (not window or row < 33 + window):
                bad[:, 64:128] = True
            if row >= 150:                              # the window still holds it
                bad[:] = True
            if row == 20:
                bad[3] = True
            assert torch.equal(torch.isnan(out[row]), bad), row


def test_prompt_tiles_deterministic(g4):
    rng = np.random.default_rng(3)
    s = Setup(g4, [(900, 200)], 1, 512, 64)
    q, out = check_attention(g4, s, 8, "f32", 0.1, 0, rng)
    for fill in (0, 0x7F):
        n = g4.kv4_attention_workspace(s.cache, s.batch, 0, 8)
        again = torch.empty_like(out)
        s.attend(q, again, 0, 0.1, 0, ws=torch.full((n,), fill, dtype=torch.uint8, device="cuda:0"))
        assert torch.equal(out, again)


@pytest.mark.parametrize("hd", [64, 512])
@pytest.mark.parametrize("span", [(0, 200), (198, 2)])
def test_attention_value_ranges(g4, hd, span):
    """Keys and values whose sizes differ by 2^20. The tiles of 128 rows hold them as fp16
    beside the largest that the tile sees, S in 2^11..2^12 a scale of it: an operand
    c S 2^-17 is rounded twice (its offset 8 S too) by 2^-25 at most, that is c S by 2^-7,
    and the largest value is 7 * 2^11 at least: 2^-7 / (7 * 2^11) < 2^-20 of it."""
    rng = np.random.default_rng(hd)
    s = Setup(g4, [(0, 200)], 1, hd, 64)
    size = torch.exp2(-torch.from_numpy(rng.integers(0, 15, 200).astype(np.float32)))
    size[180] = 64.0                                    # the first 180 rows do not see it
    k, v = (tensors(rng, 200, 1, hd, torch.float32) * size.to("cuda:0")[:, None, None] for _ in range(2))
    s.write(k, v, 0)
    ks, vs = ref.stored(as64(k)), ref.stored(as64(v))
    s.spans, s.offsets, s.rows = [span], np.array([0, span[1]], np.int32), span[1]
    s.upload()
    q = tensors(rng, span[1], 8, hd, torch.float32)
    out = torch.empty_like(q)
    s.attend(q, out, 0, 0.1, 0)
    q64, got = as64(q), as64(out)
    for row in range(span[1]):
        want, mag, delta, n = ref.attention(q64[row], ks, vs, span[0] + row, 0.1, 0)
        tol = ref.tolerance(want, mag, delta, n, 2.0 ** -23)
        if span[1] > 2:
            moved = 2 * 0.1 * 2.0 ** -20 * np.abs(ks).max() * np.abs(q64[row]).sum(-1)
            tol = tol + mag * moved[:, None] + 2.0 ** -20 * np.abs(vs).max()
        assert (np.abs(got[row] - want) <= tol).all(), row


@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-30])
def test_attention_scales(g4, scale):
    """A softmax scale of 0 (every visible key alike), a negative one, a tiny one."""
    for spans in ([(40, 1), (7, 2)], [(40, 70)]):
        for hd, heads in ((64, 4), (512, 8)):
            check_attention(g4, Setup(g4, spans, 1, hd, 32), heads, "f32", scale, 30, np.random.default_rng(hd))


def test_attention_pages_missing(g4):
    """Keys on missing pages are not seen; a row with none of its pages gives 0."""
    s = Setup(g4, [(100, 1), (20, 3), (90, 40)], 1, 256, 16)
    s.table[0, 2] = -1
    s.table[0, 6] = s.pages + 3
    s.table[1, :] = -1
    s.table[2, :4] = 2 ** 31 - 1
    s.upload()
    check_attention(g4, s, 8, "f32", 0.1, 0, np.random.default_rng(5))


def test_attention_unwritten_neighbours(g4):
    """Slots behind the last token hold scales that read as NaN: they are never seen."""
    for hd in (64, 512):
        s = Setup(g4, [(0, 1), (16, 1), (40, 2)], 1, hd, 64, fill=0xFF)
        check_attention(g4, s, 8, "f32", 0.1, 0, np.random.default_rng(6))


@pytest.mark.parametrize("bits", [0x7F80, 0xFF80, 0x7F7F, 0xFF7F, 0xFFC0, 0x8001])
def test_attention_unwritten_scales(g4, bits):
    """Behind the last token scales of infinity, of the largest values, negative ones: never seen."""
    for hd in (64, 256, 512):
        for spans in ([(16, 1), (40, 2)], [(40, 70)], [(0, 150), (3, 9)]):
            fill = np.tile(np.array([bits], np.uint16).view(np.uint8), 17 * hd // 2)
            check_attention(g4, Setup(g4, spans, 1, hd, 64, fill=fill), 8, "f32", 0.1, 0, np.random.default_rng(6))


def test_attention_nan_stays_in_its_sequence(g4):
    s = Setup(g4, [(30, 1), (30, 1)], 1, 128, 16)
    rng = np.random.default_rng(7)
    hist = Setup.__new__(Setup)
    hist.__dict__.update(s.__dict__)
    hist.spans, hist.offsets, hist.rows = [(0, 31), (0, 31)], np.array([0, 31, 62], np.int32), 62
    hist.upload()
    k, v = tensors(rng, 62, 1, 128, torch.float32), tensors(rng, 62, 1, 128, torch.float32)
    k[3] = float("nan")
    hist.write(k, v, 0)
    q = tensors(rng, 2, 4, 128, torch.float32)
    q[1, 2, 0] = float("inf")
    out = torch.empty_like(q)
    s.attend(q, out, 0, 0.1, 0)
    assert torch.isnan(out[0]).all()
    assert torch.isfinite(out[1, [0, 1, 3]]).all() and not torch.isfinite(out[1, 2]).all()


def test_attention_positions_past_the_table(g4):
    """A row past the table's positions sees the keys that the table has."""
    s = Setup(g4, [(40, 4)], 1, 64, 16, stride=3)
    s.batch.table_stride = 2
    rng = np.random.default_rng(8)
    k = tensors(rng, 32, 1, 64, torch.float32)
    w = Setup.__new__(Setup)
    w.__dict__.update(s.__dict__)
    w.spans, w.offsets, w.rows = [(0, 32)], np.array([0, 32], np.int32), 32
    w.upload()
    w.write(k, k, 0)
    q = tensors(rng, 4, 2, 64, torch.float32)
    out = torch.empty_like(q)
    s.attend(q, out, 0, 0.3, 0)
    kk = ref.stored(as64(k))
    for i in range(4):
        want, mag, delta, n = ref.attention(as64(q)[i], kk, kk, 40 + i, 0.3, 0)
        assert n == 32 and (np.abs(as64(out)[i] - want) <= ref.tolerance(want, mag, delta, n, 2.0 ** -23)).all()


def test_attention_is_deterministic_and_needs_no_clean_workspace(g4):
    rng = np.random.default_rng(9)
    s = Setup(g4, [(3000, 1), (77, 5)], 1, 256, 64)
    q, out = check_attention(g4, s, 8, "f32", 0.1, 0, rng)
    for fill in (0, 0x7F):
        n = g4.kv4_attention_workspace(s.cache, s.batch, 0, 8)
        again = torch.empty_like(out)
        s.attend(q, again, 0, 0.1, 0, ws=torch.full((n,), fill, dtype=torch.uint8, device="cuda:0"))
        assert torch.equal(out, again)


def test_large_pool_offsets(g4):
    """Pages beyond 4 GB of the pool."""
    hd, kv, page = 512, 8, 1024
    size = g4.kv4_page_bytes(kv, hd, page)
    pages = (1 << 32) // size + 3
    pool = torch.empty(pages * size, dtype=torch.uint8, device="cuda:0")
    table = dev([[pages - 1, 0]])
    off, start = dev([0, 3]), dev([1022])
    cache = g4.Kv4Cache(pool.data_ptr(), pages, page, kv, hd)
    batch = g4.Kv4Batch(1, 3, off.data_ptr(), start.data_ptr(), table.data_ptr(), 2)
    k = tensors(np.random.default_rng(2), 3, kv, hd, torch.float32)
    ko, vo = torch.zeros_like(k), torch.zeros_like(k)
    g4.kv4_write(cache, batch, 0, k.data_ptr(), k.stride(0), k.data_ptr(), k.stride(0))
    g4.kv4_read(cache, batch, 0, ko.data_ptr(), ko.stride(0), vo.data_ptr(), vo.stride(0))
    want = ref.stored(as64(k)).astype(np.float32)
    assert np.array_equal(ko.cpu().numpy(), want) and np.array_equal(vo.cpu().numpy(), want)
    # one token whose only key lies there: its value comes out
    start2 = dev([1022])
    off2 = dev([0, 1])
    b2 = g4.Kv4Batch(1, 1, off2.data_ptr(), start2.data_ptr(), table.data_ptr(), 2)
    q = tensors(np.random.default_rng(3), 1, kv, hd, torch.float32)
    out = torch.empty_like(q)
    n = g4.kv4_attention_workspace(cache, b2, 0, kv)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda:0")
    g4.kv4_attention(cache, b2, 0, kv, q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), 0.1, 1,
                     ws.data_ptr(), n)
    assert np.allclose(out.cpu().numpy()[0], want[0], rtol=2.0 ** -15, atol=0)


def test_large_pool_offsets_prompt(g4):
    """A prompt on pages beyond 4 GB of the pool: the bits of one on a small pool's."""
    hd, kv, page, rows = 512, 8, 1024, 200
    size = g4.kv4_page_bytes(kv, hd, page)
    rng = np.random.default_rng(4)
    k, q = tensors(rng, rows, kv, hd, torch.float32), tensors(rng, rows, kv, hd, torch.float32)
    off, start = dev([0, rows]), dev([900])
    outs = []
    for pages in (3, (1 << 32) // size + 3):
        pool = torch.empty(pages * size, dtype=torch.uint8, device="cuda:0")
        table = dev([[0, pages - 1]])
        cache = g4.Kv4Cache(pool.data_ptr(), pages, page, kv, hd)
        batch = g4.Kv4Batch(1, rows, off.data_ptr(), start.data_ptr(), table.data_ptr(), 2)
        g4.kv4_write(cache, batch, 0, k.data_ptr(), k.stride(0), k.data_ptr(), k.stride(0))
        out = torch.empty_like(q)
        n = g4.kv4_attention_workspace(cache, batch, 0, kv)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda:0")
        g4.kv4_attention(cache, batch, 0, kv, q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), 0.1, 1,
                         ws.data_ptr(), n)
        outs.append(out)
    assert torch.equal(*outs) and torch.isfinite(outs[0]).all() and outs[0][-1].any()


@pytest.mark.parametrize("spans", [[(70, 2), (5, 1), (400, 1)], [(70, 200)]])
def test_streams_and_graphs(g4, spans):
    """Write, attend and read on a side stream, then the same captured and replayed on new inputs."""
    rng = np.random.default_rng(11)
    s = Setup(g4, spans, 1, 256, 64)
    hist, _ = check_attention(g4, s, 8, "f32", 0.1, 0, rng)         # fills the cache
    k, v = tensors(rng, s.rows, 1, 256, torch.float32), tensors(rng, s.rows, 1, 256, torch.float32)
    q = tensors(rng, s.rows, 8, 256, torch.float32)
    ko, vo, out = torch.empty_like(k), torch.empty_like(v), torch.empty_like(q)
    ws = torch.empty(g4.kv4_attention_workspace(s.cache, s.batch, 0, 8), dtype=torch.uint8, device="cuda:0")

    def step(st):
        s.write(k, v, 0, st)
        s.attend(q, out, 0, 0.1, 0, ws=ws, stream=st)
        s.read(ko, vo, 0, st)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    step(side.cuda_stream)
    side.synchronize()
    first = [x.clone() for x in (ko, vo, out)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream().cuda_stream)
    for x in (ko, vo, out):
        x.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, (ko, vo, out)))
    new = [tensors(rng, s.rows, n, 256, torch.float32) for n in (1, 1, 8)]
    for x, y in zip((k, v, q), new):
        x.copy_(y)
    graph.replay()
    torch.cuda.synchronize()
    replayed = [x.clone() for x in (ko, vo, out)]
    step(None)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(replayed, (ko, vo, out)))


def test_host_pointers_are_refused(g4):
    s = Setup(g4, [(0, 4)], 1, 64, 16)
    k = tensors(np.random.default_rng(0), 4, 1, 64, torch.float32)
    host = torch.empty(4096, dtype=torch.float32)
    with pytest.raises(g4.G4Error):
        g4.kv4_write(s.cache, s.batch, 0, host.data_ptr() // 16 * 16 + 16, 64, k.data_ptr(), 64)
    bad = g4.Kv4Batch(1, 4, host.data_ptr() // 16 * 16 + 16, s.d_start.data_ptr(), s.d_table.data_ptr(), 1)
    with pytest.raises(g4.G4Error):
        g4.kv4_read(s.cache, bad, 0, k.data_ptr(), 64, k.data_ptr(), 64)


# ---------------------------------------------------------------------------
# reordering

def reorder_ref(tables, spare, parents, lengths, page, pools):
    """The definition, on copies."""
    groups, beams = parents.shape
    out_t, out_s, pools = tables.copy(), spare.copy(), [p.copy() for p in pools]
    old = [p.copy() for p in pools]
    for g in range(groups):
        full, left = divmod(int(lengths[g]), page)
        for w in range(beams):
            i = g * beams + w
            p = g * beams + int(parents[g, w]) if 0 <= parents[g, w] < beams else i
            out_t[i, :full] = tables[p, :full]
            if p != i and left and full < tables.shape[1]:
                out_t[i, full], out_s[i] = spare[i], tables[i, full]
                n = -(-left // 16)
                for a, b in zip(pools, old):
                    a[spare[i], :, :n] = b[tables[p, full], :, :n]
    return out_t, out_s, pools


@pytest.mark.parametrize("groups,beams,page,lengths", [(1, 4, 16, [5]), (2, 3, 32, [64, 33]), (3, 8, 64, [0, 200, 63]),
                                                       (1, 1, 16, [40]), (2, 32, 16, [17, 31])])
def test_reorder(g4, groups, beams, page, lengths):
    rng = np.random.default_rng(beams)
    stride = max(lengths) // page + 2
    rows = groups * beams
    shapes = [(1, 256), (2, 64), (1, 512)]
    pages = rows * (stride + 1)
    ids = rng.permutation(pages).astype(np.int32)
    tables, spare = ids[:rows * stride].reshape(rows, stride), ids[rows * stride:]
    pools = [rng.integers(0, 256, (pages, kv, page // 16, 17 * hd), dtype=np.uint8) for kv, hd in shapes]
    d = [dev(p, torch.uint8) for p in pools]
    parents = rng.integers(0, beams, (groups, beams)).astype(np.int32)
    parents[0, 0] = -3 if beams > 1 else 9          # counts as the beam itself
    t_out, s_out = torch.empty((rows, stride), dtype=torch.int32, device="cuda:0"), torch.empty(
        rows, dtype=torch.int32, device="cuda:0")
    caches = g4.kv4_caches([g4.Kv4Cache(x.data_ptr(), pages, page, kv, hd) for x, (kv, hd) in zip(d, shapes)])
    d_par, d_len, d_t, d_s = dev(parents), dev(lengths), dev(tables), dev(spare)
    want = reorder_ref(tables, spare, parents, lengths, page, pools)
    for _ in range(2):                               # the same call again gives the same
        g4.kv4_reorder(caches, groups, beams, d_par.data_ptr(), d_len.data_ptr(), d_t.data_ptr(), t_out.data_ptr(),
                       stride, d_s.data_ptr(), s_out.data_ptr())
        assert np.array_equal(t_out.cpu().numpy(), want[0]) and np.array_equal(s_out.cpu().numpy(), want[1])
        assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(d, want[2]))


def test_reorder_bad_pages(g4):
    """Page numbers outside the pool: the tables follow, no page is touched."""
    pool = torch.arange(4 * 17 * 64, dtype=torch.int64, device="cuda:0").to(torch.uint8)
    before = pool.clone()
    table = dev([[9, -1], [-4, 1]])
    spare, parents, lengths = dev([77, -2]), dev([1, 0]), dev([5])
    t_out, s_out = torch.empty_like(table), torch.empty_like(spare)
    g4.kv4_reorder(g4.kv4_caches([g4.Kv4Cache(pool.data_ptr(), 4, 16, 1, 64)]), 1, 2, parents.data_ptr(),
                   lengths.data_ptr(), table.data_ptr(), t_out.data_ptr(), 2, spare.data_ptr(), s_out.data_ptr())
    assert t_out.tolist() == [[77, -1], [-2, 1]] and s_out.tolist() == [9, -4]
    assert torch.equal(pool, before)
    # lengths past the table, and negative ones
    for n in (1000, -5):
        g4.kv4_reorder(g4.kv4_caches([g4.Kv4Cache(pool.data_ptr(), 4, 16, 1, 64)]), 1, 2, parents.data_ptr(),
                       dev([n]).data_ptr(), table.data_ptr(), t_out.data_ptr(), 2, spare.data_ptr(), s_out.data_ptr())
        assert torch.equal(pool, before)
        assert s_out.tolist() == [77, -2]


@pytest.mark.parametrize("missing", [-1, 77])
def test_reorder_of_a_missing_page(g4, missing):
    """The parent's part-full page is no page: its tokens are not seen by the child either,
    whatever the child's spare page held before."""
    page, hd, length = 16, 64, 20
    rng = np.random.default_rng(3)
    pool = dev(rng.integers(0, 256, (8, 1, 1, 17 * hd)), torch.uint8)
    cache = g4.Kv4Cache(pool.data_ptr(), 8, page, 1, hd)
    table, spare = dev([[0, missing, 5], [1, 2, 6], [3, 7, 6]]), dev([3, 4, 5])
    off, start = dev([0, length, 2 * length, 3 * length]), dev([0, 0, 0])
    k = tensors(rng, 3 * length, 1, hd, torch.float32)
    batch = g4.Kv4Batch(3, 3 * length, off.data_ptr(), start.data_ptr(), table.data_ptr(), 3)
    g4.kv4_write(cache, batch, 0, k.data_ptr(), k.stride(0), k.data_ptr(), k.stride(0))
    before = pool.clone()
    parents, lengths = dev([0, 0, 1]), dev([length])
    t_out, s_out = torch.empty_like(table), torch.empty_like(spare)
    g4.kv4_reorder(g4.kv4_caches([cache]), 1, 3, parents.data_ptr(), lengths.data_ptr(), table.data_ptr(),
                   t_out.data_ptr(), 3, spare.data_ptr(), s_out.data_ptr())
    assert t_out.tolist() == [[0, missing, 5], [0, missing, 6], [1, 5, 6]] and s_out.tolist() == [3, 4, 7]
    want = before.clone()
    want[5] = before[2]                                # only the beam whose parent has its page copies one
    assert torch.equal(pool, want)
    # the child sees what the parent sees: the 16 keys of the full page
    q = tensors(rng, 1, 1, hd, torch.float32).expand(3, 1, hd).contiguous()
    out = torch.empty_like(q)
    step, at = dev([0, 1, 2, 3]), dev([length - 1] * 3)
    b = g4.Kv4Batch(3, 3, step.data_ptr(), at.data_ptr(), t_out.data_ptr(), 3)
    ws = torch.empty(g4.kv4_attention_workspace(cache, b, 0, 1), dtype=torch.uint8, device="cuda:0")
    g4.kv4_attention(cache, b, 0, 1, q.data_ptr(), hd, out.data_ptr(), hd, 0.1, 0, ws.data_ptr(), ws.numel())
    kk = ref.stored(as64(k[:16]))
    want, mag, delta, n = ref.attention(as64(q)[0], kk, kk, 15, 0.1, 0)
    tol = ref.tolerance(want, mag, delta, n, 2.0 ** -23)
    assert (np.abs(as64(out)[0] - want) <= tol).all() and torch.equal(out[0], out[1])
    assert not torch.equal(out[0], out[2])


@pytest.mark.parametrize("hd,kv,heads,name", [(512, 1, 8, "f32"), (128, 4, 16, "bf16")])
def test_attention_in_a_workspace_of_the_largest_call(g4, hd, kv, heads, name):
    """One buffer, sized for the largest call, serves chunks, single tokens and shorter tables
    with the bits that they have in their own; nothing behind what a call asked for is touched."""
    rng = np.random.default_rng(12)
    big = Setup(g4, [(0, 600)] * 3, kv, hd, 64, stride=64)
    n = g4.kv4_attention_workspace(big.cache, big.batch, kind_of(g4, name), heads)
    ws = torch.empty(n + 4096, dtype=torch.uint8, device="cuda:0")
    for spans, stride in (([(900, 1)], None), ([(2900, 70)], None), ([(100, 90)], None), ([(50, 1), (700, 300), (3, 1)], 64),
                          ([(0, 500)] * 3, 64)):
        s = Setup(g4, spans, kv, hd, 64, stride=stride)
        q, want = check_attention(g4, s, heads, name, 0.1, 0, rng)
        need = g4.kv4_attention_workspace(s.cache, s.batch, kind_of(g4, name), heads)
        assert need <= n
        ws.fill_(0x5A)
        out = torch.empty_like(want)
        s.attend(q, out, kind_of(g4, name), 0.1, 0, ws=ws[:n])
        assert torch.equal(out, want) and (ws[need:] == 0x5A).all()


@pytest.mark.parametrize("hd,kv", [(128, 2), (256, 1), (512, 1)])
@pytest.mark.parametrize("start", [0, 700])
def test_prompt_tiles_groups_of_different_sizes(g4, hd, kv, start):
    """Values whose groups of dimensions differ by up to 2^30: every group as exact as if it
    were alone (the bound is the dimension's own)."""
    rng = np.random.default_rng(hd + start)
    rows = 150
    s = Setup(g4, [(0, start + rows)], kv, hd, 64)
    size = np.repeat(2.0 ** -np.array([0, 9, 18, 30, 14, 27, 5, 22][:hd // 64] * kv, np.float32), 64).reshape(kv, hd)
    size[kv - 1] = size[kv - 1][::-1]                   # not the same in every head
    k = tensors(rng, start + rows, kv, hd, torch.float32)
    v = (tensors(rng, start + rows, kv, hd, torch.float32) * dev(size, torch.float32)).contiguous()
    s.write(k, v, 0)
    ks, vs = ref.stored(as64(k)), ref.stored(as64(v))
    s.spans, s.offsets, s.rows = [(start, rows)], np.array([0, rows], np.int32), rows
    s.upload()
    for name in ("f32", "bf16"):
        q = tensors(rng, rows, 8, hd, TYPES[name])
        out = torch.empty_like(q)
        s.attend(q, out, kind_of(g4, name), 0.1, 0)
        q64, got = as64(q), as64(out)
        for row in range(rows):
            want, mag, delta, n = ref.attention(q64[row], ks, vs, start + row, 0.1, 0)
            tol = ref.tolerance(want, mag, delta, n, torch.finfo(TYPES[name]).eps)
            assert (np.abs(got[row] - want) <= tol).all(), (name, row)
