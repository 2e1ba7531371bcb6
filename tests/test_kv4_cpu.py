"""The 4-bit cache and beam search on the CPU: sizes and refusals (every bad
argument is refused before any GPU work), and the reference's own layout."""

import numpy as np
import pytest

import kv4_ref as ref

P = 0x10000          # an aligned address that no refused call may touch


def cache(g4, **kw):
    d = dict(pages=P, num_pages=4, page_size=64, kv_heads=1, head_dim=256)
    d.update(kw)
    return g4.Kv4Cache(**d)


def batch(g4, **kw):
    d = dict(n=2, rows=8, offsets=P, start_pos=P, page_table=P, table_stride=4)
    d.update(kw)
    return g4.Kv4Batch(**d)


BAD_CACHE = [dict(pages=None), dict(pages=P + 8), dict(num_pages=0), dict(page_size=24), dict(page_size=8),
             dict(page_size=2048), dict(page_size=0), dict(kv_heads=0), dict(kv_heads=257), dict(head_dim=96),
             dict(head_dim=0), dict(head_dim=1024)]
BAD_BATCH = [dict(n=-1), dict(n=65537), dict(rows=-1), dict(rows=(1 << 22) + 1), dict(offsets=None),
             dict(start_pos=None), dict(page_table=None), dict(offsets=P + 2), dict(page_table=P + 1),
             dict(table_stride=0),
             dict(table_stride=(1 << 24) + 1)]


def test_page_bytes(g4):
    assert g4.kv4_page_bytes(1, 256, 64) == 64 // 16 * 17 * 256
    assert g4.kv4_page_bytes(8, 128, 16) == 8 * 17 * 128
    for bad in ((0, 64, 64), (1, 65, 64), (1, 64, 48), (1, 64, 8), (300, 64, 64)):
        assert g4.kv4_page_bytes(*bad) == 0


@pytest.mark.parametrize("name", ["g4_kv4_write", "g4_kv4_read"])
def test_move_refusals(g4, name):
    f = getattr(g4.load(), name)

    def call(c=None, b=None, kind=0, k=P, ks=256, v=P, vs=256):
        return f(c or cache(g4), b or batch(g4), kind, k, ks, v, vs, None)
    for kw in BAD_CACHE:
        assert call(c=cache(g4, **kw)) == -1, kw
    for kw in BAD_BATCH:
        assert call(b=batch(g4, **kw)) == -1, kw
    for kw in (dict(kind=3), dict(kind=-1), dict(k=None), dict(v=None), dict(k=P + 4), dict(ks=255), dict(vs=258),
               dict(ks=-256), dict(kind=1, ks=260), dict(ks=1 << 50)):
        assert call(**kw) == -1, kw
    assert f(None, batch(g4), 0, P, 256, P, 256, None) == -1
    assert f(cache(g4), None, 0, P, 256, P, 256, None) == -1
    # nothing to do: no GPU work
    assert call(b=batch(g4, n=0)) == 0 and call(b=batch(g4, rows=0)) == 0


def test_attention_refusals(g4):
    f = g4.load().g4_kv4_attention

    def call(c=None, b=None, kind=0, heads=8, q=P, qs=2048, o=P, os=2048, scale=1.0, window=0, ws=P, wb=1 << 40):
        return f(c or cache(g4), b or batch(g4), kind, heads, q, qs, o, os, scale, window, ws, wb, None)
    for kw in BAD_CACHE:
        assert call(c=cache(g4, **kw)) == -1, kw
    for kw in BAD_BATCH:
        assert call(b=batch(g4, **kw)) == -1, kw
    for kw in (dict(kind=9), dict(heads=0), dict(heads=-8), dict(c=cache(g4, kv_heads=3)), dict(heads=65, qs=65 * 256),
               dict(q=None), dict(o=None), dict(q=P + 2), dict(qs=2047), dict(os=2050), dict(scale=float("nan")),
               dict(scale=float("inf")), dict(window=-1), dict(ws=None), dict(ws=P + 8), dict(wb=0)):
        assert call(**kw) == -1, kw
    assert call(b=batch(g4, n=0)) == 0 and call(b=batch(g4, rows=0)) == 0
    with pytest.raises(g4.G4Error):
        g4.kv4_attention_workspace(cache(g4), batch(g4), 0, 7 * 64 + 1 + 64)
    assert g4.kv4_attention_workspace(cache(g4), batch(g4), 0, 8) > 0


def prompt_bytes(hd, kv, heads, f32, n, rows, length):
    """What the tiles of 128 rows fill for such a call: per row tile and kv head, for as many key
    ranges as the rounds of the grid ask for, an output of 128 rows, their maxima and sums."""
    group, room = heads // kv, 74 if hd > 256 else 148
    tokens = 128 // group
    items, tiles = -(-rows // tokens) * kv, -(-length // 64)
    best, splits = None, 1
    for s in range(1, min(32, tiles) + 1):
        if s > 1 and items * s > 4 * room:
            break
        cost = -(-items * s // room) * (tiles / s + 3) + (items * s * hd / 20000 if s > 1 else 0)
        if best is None or cost < 0.97 * best:
            best, splits = cost, s
    if splits == 1 and tiles <= (16 if f32 else 256):
        return 0
    return (rows // tokens + n) * kv * splits * 128 * (hd + 2) * 4


@pytest.mark.parametrize("hd,kv,heads", [(64, 1, 8), (128, 8, 32), (128, 2, 10), (256, 1, 8), (512, 1, 8), (512, 2, 4)])
@pytest.mark.parametrize("kind", [0, 1])
def test_attention_workspace_serves_every_smaller_call(g4, kind, hd, kv, heads):
    """A buffer sized for the longest prompt, the most sequences and the longest table is enough
    for every decode step, shorter prompt and table, and holds what their plan fills."""
    sizes = [(n, rows, stride) for n in (1, 2, 5, 16, 64) for rows in (1, 8, 60, 63, 70, 75, 100, 512, 513, 4096, 20000)
             for stride in (1, 16, 17, 256, 2048)]
    c = cache(g4, kv_heads=kv, head_dim=hd)
    need = {s: g4.kv4_attention_workspace(c, batch(g4, n=s[0], rows=s[1], table_stride=s[2]), kind, heads)
            for s in sizes}
    slots = {64: 592, 128: 592, 256: 592, 512: 296}[hd] * 8 * (hd + 2) * 4
    for s, b in need.items():
        assert b >= slots, s                            # the few rows' partial outputs, two for every CTA
        if s[1] * (heads // kv) >= (576 if hd >= 256 and s[0] * kv < 4 else 112) * s[0]:
            assert b >= prompt_bytes(hd, kv, heads, kind == 0, s[0], s[1], s[2] * 64), s
        assert b == max(m for t, m in need.items() if all(x <= y for x, y in zip(t, s))), s


def test_beam_refusals(g4):
    f = g4.load().g4_beam_select

    def call(g=1, w=4, v=1000, kind=0, x=P, xs=1000, s=P, fin=None, eos=-1, os=P, pa=P, to=P, fo=None, ws=P,
             wb=1 << 40):
        return f(g, w, v, kind, x, xs, s, fin, eos, os, pa, to, fo, ws, wb, None)
    for kw in (dict(g=-1), dict(g=65537), dict(w=0), dict(w=33), dict(v=0), dict(v=(1 << 24) + 1), dict(kind=3),
               dict(x=None), dict(x=P + 2), dict(kind=1, x=P + 1), dict(xs=999), dict(s=None), dict(s=P + 2),
               dict(eos=1000), dict(fin=P), dict(os=None), dict(pa=None), dict(to=None), dict(ws=None),
               dict(ws=P + 4), dict(wb=8)):
        assert call(**kw) == -1, kw
    assert call(g=0) == 0
    for bad in ((1, 0, 10), (1, 33, 10), (1, 4, 0), (-1, 4, 10)):
        assert g4.load().g4_beam_workspace(*bad) == 0
        with pytest.raises(g4.G4Error):
            g4.beam_workspace(*bad)


def test_beam_workspace_serves_every_smaller_call(g4):
    """A buffer sized for the largest search is enough when searches end, beams are fewer or the
    vocabulary is shorter, and it holds what a call of those sizes fills: 16 bytes and a
    key of 8 per beam for every slice of a row, as many slices as four CTAs on each of
    148 SMs leave it."""
    sizes = [(g, w, v) for g in (1, 2, 3, 7, 16, 64, 65, 200) for w in (1, 2, 4, 5, 8, 31, 32)
             for v in (1, 4096, 4097, 50001, 100000, 262144)]
    need = {s: g4.beam_workspace(*s) for s in sizes}
    for s, n in need.items():
        rows, chunks = s[0] * s[1], -(-s[2] // 4096)
        slices = 592 // rows
        per = chunks if slices <= 1 else -(-chunks // slices)
        assert n >= rows * -(-chunks // per) * (16 + 8 * s[1]), s
        smaller = [m for t, m in need.items() if all(a <= b for a, b in zip(t, s))]
        assert max(smaller) == n, s
    refused = g4.load().g4_beam_select
    n = g4.beam_workspace(3, 4, 262144)
    args = (P, 262144, P, None, -1, P, P, P, None, P)
    assert refused(3, 4, 262144, 0, *args, n - 1, None) == -1


def test_reorder_refusals(g4):
    f = g4.load().g4_kv4_reorder
    far = P + (1 << 20)

    def call(caches=None, layers=None, g=2, w=4, pa=P, le=P, ti=P, to=far, stride=4, si=P, so=far):
        cs = g4.kv4_caches(caches or [cache(g4), cache(g4, head_dim=512)])
        return f(cs, len(cs) if layers is None else layers, g, w, pa, le, ti, to, stride, si, so, None)
    for kw in BAD_CACHE:
        assert call(caches=[cache(g4), cache(g4, **kw)]) == -1, kw
    for kw in (dict(caches=[cache(g4), cache(g4, page_size=32)]), dict(caches=[cache(g4), cache(g4, num_pages=5)]),
               dict(layers=0), dict(layers=65), dict(g=-1), dict(g=65537), dict(w=0), dict(w=33), dict(pa=None),
               dict(le=None), dict(ti=None), dict(to=None), dict(si=None), dict(so=None), dict(to=P), dict(so=P),
               dict(to=P + 4 * 4 * 8 - 4), dict(so=P + 4 * 8 - 4), dict(stride=0), dict(pa=P + 2)):
        assert call(**kw) == -1, kw
    assert call(g=0) == 0


def test_outputs_over_inputs_are_refused(g4):
    """Outputs that share a byte with an input: refused; next to it: not."""
    f, r = g4.load().g4_beam_select, g4.load().g4_kv4_reorder

    def beam(**kw):
        a = dict(s=P, fin=P + 0x100, os=P + 0x200, pa=P + 0x300, to=P + 0x400, fo=P + 0x500) | kw
        return f(2, 4, 1000, 0, P + 0x1000, 1000, a["s"], a["fin"], 3, a["os"], a["pa"], a["to"], a["fo"], P, 1 << 40,
                 None)

    def reorder(**kw):
        a = dict(pa=P, le=P + 0x100, ti=P + 0x200, to=P + 0x400, si=P + 0x600, so=P + 0x700) | kw
        return r(g4.kv4_caches([cache(g4)]), 1, 2, 4, a["pa"], a["le"], a["ti"], a["to"], 4, a["si"], a["so"], None)
    for kw in (dict(os=P), dict(os=P + 28), dict(os=P - 28), dict(pa=P + 0x100 + 4), dict(to=P + 4), dict(fo=P + 0x100),
               dict(fo=P + 0x100 + 7), dict(fo=P + 31)):
        assert beam(**kw) == -1, kw
    for kw in (dict(to=P), dict(to=P + 0x600 - 124), dict(so=P + 0x200 + 124), dict(so=P + 28), dict(so=P + 0x104),
               dict(to=P + 0x200), dict(so=P + 0x600), dict(to=P + 0x100 + 4)):
        assert reorder(**kw) == -1, kw
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():                   # the addresses are nobody's
        for kw in (dict(), dict(os=P + 32), dict(fo=P + 0x100 + 8)):
            assert beam(**kw) != -1, kw
        for kw in (dict(), dict(so=P + 32), dict(to=P + 0x200 + 128)):
            assert reorder(**kw) != -1, kw


def test_reference_layout_is_a_bijection():
    """Every nibble and scale of a record belongs to one token and dimension."""
    rng = np.random.default_rng(0)
    for hd in (64, 256):
        c = ref.Cache(1, 16, 1, hd, fill=0)
        seen = np.zeros(17 * hd, np.int64)
        for t in range(16):
            c.bytes[:] = 0
            x = rng.standard_normal(hd) + 0.1
            c.put(0, t, 0, x, x)
            seen += c.bytes[0, 0, 0] != 0
        assert (seen > 0).all() and (seen <= 2).all()


def test_reference_rounding():
    """Ties to even, exact next to a border, special groups."""
    x = np.zeros((5, 64))
    x[0, :4] = [7, 0.5, 1.5, -2.5]                     # scale 1: 0, 2, -2
    x[1, :2] = [7, np.nextafter(np.float32(0.5), np.float32(1))]
    x[2, 3] = np.inf
    x[3, 5] = 2.0 ** -101
    x[4, 0] = np.nan
    c, s = ref.quantise(x)
    assert c[0, :4].tolist() == [7, 0, 2, -2] and c[1, 1] == 1
    assert np.isnan(s[2, 0]) and np.isnan(s[4, 0]) and s[3, 0] == 0 and not c[2:].any()


def test_no_gpu_is_an_error(g4):
    """Valid arguments without a GPU: an error code, no abort."""
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("has a GPU")
    L = g4.load()
    assert L.g4_kv4_write(cache(g4), batch(g4), 0, P, 256, P, 256, None) in (-1, -3)
