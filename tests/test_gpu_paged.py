"""The operators over a paged cache (attention_paged, kv_append_paged, qk_norm_rope) against their definitions in 64 bits.

Tolerances.  u = half a step of the type (bf16 2^-8, f16 2^-11, f32 2^-24), e = 2^-24.
  * attention: the result is rounded once (u), the probabilities are rounded to the type before the second product (u, of
    each term p v, so of sum p |v| / sum p =: A), and a score is a sum of dh products in f32 (at most (dh + 8) e of
    S = scale * sum |q| |k|, which moves a probability by as much, in the numerator and in the sum); 2^-20 of A for the
    exponentials and the sums over keys: |o - o64| <= (2 u + 2 (dh + 8) e S + 2^-20) A.
  * rotation: one rounding (u), sine and cosine to 2^-22, products and their sum: u |y| + 2^-20 (|a| + |b|) for the pair.
  * norm: a sum of dh squares ((dh / 2 + 8) e of the normalised row), then the rotation.
f16 results below 2^-14 are rounded in steps of 2^-24: 2^-25 more.
"""
import ctypes

import numpy as np
import pytest

import ophip
from ophip import TensorLayout, dt

pytestmark = pytest.mark.gpu

HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
CODE = {"f16": dt.F16, "bf16": dt.BF16, "f32": dt.F32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
E = 2.0 ** -24


def encode(x, kind):
    """f64 values rounded to the type, as the bits that are uploaded."""
    x = np.asarray(x, np.float32)
    if kind == "f16":
        return x.astype(np.float16)
    if kind == "f32":
        return x
    b = np.ascontiguousarray(x).view(np.uint32)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r).astype(np.uint16)


def decode(bits, kind):
    if kind == "bf16":
        return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return bits.astype(np.float64)


def store(kind):
    return {"f16": np.float16, "bf16": np.uint16, "f32": np.float32}[kind]


def layout(view, kind):
    return TensorLayout(CODE[kind], view.shape, view.strides)


class Buffer:
    """A host array and its copy on the device; `view(x)`: the layout and address of a numpy view of it."""

    def __init__(self, gpu, array, kind=None):
        self.gpu, self.host, self.kind = gpu, np.ascontiguousarray(array), kind
        self.mem = gpu.from_host(self.host)

    def view(self, x=None):
        x = self.host if x is None else x
        off = x.__array_interface__["data"][0] - self.host.__array_interface__["data"][0] if x.size else 0
        code = CODE[self.kind] if self.kind else {np.dtype(np.uint32): dt.U32, np.dtype(np.int32): dt.I32, np.dtype(np.uint64): dt.U64, np.dtype(np.int64): dt.I64}[x.dtype]
        return TensorLayout(code, x.shape, x.strides), self.mem.ptr + off

    def back(self, stream):
        return self.gpu.to_host(self.mem, self.host.dtype, self.host.size, stream=stream).reshape(self.host.shape)


class Batch:
    """A paged cache and a packed batch: lens = [(new tokens, keys)], `pad` tokens behind them."""

    def __init__(self, gpu, rng, kind, nh, nkvh, dh, page, lens, pad=0, spare=2, junk=np.nan, token_major=False, head_gap=0):
        self.kind, self.nh, self.nkvh, self.dh, self.page, self.lens = kind, nh, nkvh, dh, page, lens
        self.start = np.concatenate([[0], np.cumsum([n for n, _ in lens])]).astype(np.uint32)
        self.nt = int(self.start[-1]) + pad
        used = [-(-l // page) for _, l in lens]
        npages, cols = sum(used) + spare, max(1, max(used))
        order = rng.permutation(npages)
        table, at = np.full((len(lens), cols), 0xFFFFFFFF, np.uint32), 0
        for s, c in enumerate(used):
            table[s, :c] = order[at:at + c]
            at += c
        shape = (npages, page, nkvh, dh + head_gap) if token_major else (npages, nkvh, page, dh + head_gap)
        cache = [np.full(shape, junk, np.float64) for _ in range(2)]
        views = [(c.swapaxes(1, 2) if token_major else c)[..., :dh] for c in cache]
        for s, (_, l) in enumerate(lens):
            for j in range(l):
                for v in views:
                    v[table[s, j // page], :, j % page] = rng.standard_normal((nkvh, dh))
        self.cache = [Buffer(gpu, encode(c, kind), kind) for c in cache]
        self.cache_views = [(c.host.swapaxes(1, 2) if token_major else c.host)[..., :dh] for c in self.cache]
        self.table, self.q_start = Buffer(gpu, table), Buffer(gpu, self.start)
        self.kv_len = Buffer(gpu, np.array([l for _, l in lens], np.uint32))
        self.q = Buffer(gpu, encode(rng.standard_normal((self.nt, nh, dh)) * 1.5, kind), kind)
        self.o = Buffer(gpu, encode(np.full((self.nt, nh, dh), 0.125), kind), kind)

    def batch_args(self):
        return self.table.view() + self.q_start.view() + self.kv_len.view()

    def cache_args(self):
        return self.cache[0].view(self.cache_views[0]) + self.cache[1].view(self.cache_views[1])

    def args(self, mask, scale=None):
        scale = self.dh ** -0.5 if scale is None else scale
        q, o = self.q.host.transpose(1, 0, 2), self.o.host.transpose(1, 0, 2)
        return ophip.AttentionPagedArgs(*self.q.view(q), *self.cache_args(), *self.o.view(o), *self.batch_args(), mask, scale)

    def keys(self, s, which, cache=None):
        l = self.lens[s][1]
        views = self.cache_views if cache is None else cache
        rows = [views[which][self.table.host[s, j // self.page], :, j % self.page] for j in range(l)]
        return decode(np.array(rows).reshape(l, self.nkvh, self.dh), self.kind)

    def expected(self, mask, scale=None, q=None, cache=None):
        """(o in 64 bits, tolerance); rows of no sequence as they were, tolerance 0."""
        scale = float(np.float32(self.dh ** -0.5 if scale is None else scale))
        q = decode(self.q.host, self.kind) if q is None else q
        o, tol = decode(self.o.host, self.kind), np.zeros((self.nt, self.nh, self.dh))
        u, group = HALF[self.kind], self.nh // self.nkvh
        for s, (n, l) in enumerate(self.lens):
            k, v = self.keys(s, 0, cache), self.keys(s, 1, cache)
            for i in range(n):
                t, keep = self.start[s] + i, min(l, max(0, l - n + i + 1)) if mask else l
                for h in range(self.nh):
                    if keep == 0:
                        o[t, h], tol[t, h] = 0, 0
                        continue
                    kk, vv = k[:keep, h // group], v[:keep, h // group]
                    x = kk @ q[t, h] * scale
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    o[t, h] = p @ vv
                    big = (np.abs(kk) @ np.abs(q[t, h])).max() * abs(scale)
                    tol[t, h] = (2 * u + 2 * (self.dh + 8) * E * big + 2.0 ** -20) * (p @ np.abs(vv)) + 2.0 ** -25
        return o, tol


def check(got, want, tol, what=""):
    """Within the tolerance, and not finite exactly where the definition is not."""
    fine = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fine), what
    off = np.where(fine, np.abs(np.where(fine, got, 0) - np.where(fine, want, 0)) - np.where(fine, tol, 0), 0)
    assert (off <= 0).all(), "%s: %d of %d beyond their tolerance, worst by %g at %s" % (
        what, (off > 0).sum(), off.size, off.max(), np.unravel_index(np.argmax(off), off.shape))


def run(gpu, stream, args, op=None, workspace=True):
    op = op or ophip.AttentionPaged(gpu)
    need = op.scheme(args, 1 << 40)
    ws = gpu.malloc(need) if need and workspace else None
    op.launch(args, ws, stream)
    stream.synchronize()
    return ws


def attend(gpu, stream, b, mask, **kw):
    run(gpu, stream, b.args(mask, kw.pop("scale", None)), **kw)
    return decode(b.o.back(stream), b.kind)


def _many_sequences(count, seed):
    rng = np.random.default_rng(seed)
    lens = [(1, int(l)) for l in rng.integers(1, 60, count)]
    for i in rng.integers(0, count, 4):
        lens[i] = (int(rng.integers(2, 30)), 400)
    lens[count // 2] = (0, 20)
    return lens


@pytest.mark.parametrize("count", [63, 64, 65, 300, 600])
@pytest.mark.parametrize("group", [2, 20])
def test_attention_paged_many_sequences(gpu, stream, count, group):
    """More sequences than lanes of a wave and than threads of a workgroup: each finds its work in the prefix sums."""
    b = Batch(gpu, np.random.default_rng(16), "f16", group, 1, 64, 16, _many_sequences(count, count), pad=2)
    want, tol = b.expected(1)
    check(attend(gpu, stream, b, 1), want, tol)


SHAPES = [  # nh, nkvh, dh, page, lens
    (4, 4, 64, 16, [(1, 1)]),
    (4, 1, 64, 16, [(1, 33), (1, 16), (1, 0), (1, 300)]),
    (8, 2, 128, 7, [(1, 5), (1, 129), (1, 640)]),
    (7, 1, 128, 32, [(1, 1000)]),
    (16, 1, 64, 1, [(1, 77), (1, 257)]),
    (20, 1, 128, 24, [(1, 200), (2, 31)]),
    (6, 3, 64, 24, [(5, 5), (0, 40), (3, 50), (9, 9)]),
    (4, 4, 128, 64, [(70, 70), (3, 200)]),
    (2, 2, 64, 128, [(130, 400)]),
    (8, 2, 128, 16, [(33, 33), (65, 130), (1, 17)]),
    (3, 1, 64, 256, [(150, 150)]),
    (12, 4, 64, 100, [(40, 700), (1, 900), (2, 3)]),
    (24, 1, 128, 48, [(11, 95)]),
    (4, 2, 128, 16, [(10, 4), (6, 0), (3, 3)]),  # fewer keys than tokens: rows that see nothing
    (2, 1, 40, 16, [(3, 50)]),                     # a head dimension of no matrix kernel
    (2, 2, 8, 5, [(4, 21), (1, 7)]),
    (1, 1, 1, 3, [(2, 9)]),
]


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("mask", [1, 0])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%d-%d-%d-%d-%s" % (s[0], s[1], s[2], s[3], "_".join("%dof%d" % x for x in s[4])))
def test_attention_paged(gpu, stream, shape, mask, kind):
    rng = np.random.default_rng(7)
    b = Batch(gpu, rng, kind, *shape[:4], shape[4], pad=3)
    want, tol = b.expected(mask)
    check(attend(gpu, stream, b, mask), want, tol)
    assert np.array_equal(b.q.back(stream).view(np.uint8), b.q.host.view(np.uint8))  # q is read only
    for c in b.cache:
        assert np.array_equal(c.back(stream).view(np.uint8), c.host.view(np.uint8))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("lens", [[(1, 3000)], [(1, 3000), (1, 10), (1, 700)], [(40, 2500)], [(16, 1500), (1, 5), (90, 90)]], ids=str)
def test_attention_paged_keys_split_over_workgroups(gpu, stream, lens, kind):
    """Few rows and many keys: a tile's keys go to several workgroups and are joined; with the workspace that scheme
    reports, and with one from the queue's allocator."""
    rng = np.random.default_rng(8)
    b = Batch(gpu, rng, kind, 4, 1, 128, 32, lens)
    want, tol = b.expected(1)
    one = attend(gpu, stream, b, 1)
    check(one, want, tol)
    b.o.gpu.upload(b.o.mem, b.o.host)
    two = attend(gpu, stream, b, 1, workspace=False)
    assert np.array_equal(one, two)  # the same bits


@pytest.mark.parametrize("tile", ["0", "1", "2"])
@pytest.mark.parametrize("mask", [1, 0])
@pytest.mark.parametrize("lens", [[(1, 700), (3, 9), (0, 5)], [(300, 330)], [(17, 400), (1, 1500), (40, 40)], [(1100, 1100)], [(5, 2)] + [(1, 30)] * 66 + [(30, 600)]],
                         ids=["decode", "prompt", "mixed", "long", "many"])
@pytest.mark.parametrize("dh", [64, 128])
def test_attention_paged_every_size_of_tile(gpu, stream, monkeypatch, tile, lens, mask, dh):
    """Each kernel on every kind of batch, also those that another would be chosen for."""
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
    b = Batch(gpu, np.random.default_rng(17), "f16", 2, 1, dh, 24, lens, pad=1)
    want, tol = b.expected(mask)
    check(attend(gpu, stream, b, mask), want, tol)


@pytest.mark.parametrize("tile", ["1", "2"])
@pytest.mark.parametrize("slots", ["3", "40"])
def test_attention_paged_few_and_many_key_ranges(gpu, stream, monkeypatch, tile, slots):
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
    monkeypatch.setenv("OPHIP_ATTN_PAGED_SLOTS", slots)
    b = Batch(gpu, np.random.default_rng(18), "bf16", 4, 2, 64, 16, [(20, 2000), (1, 3000), (70, 900)])
    want, tol = b.expected(1)
    check(attend(gpu, stream, b, 1), want, tol)


@pytest.mark.parametrize("shape", [(4, 2, 64, 16, [(1, 90), (1, 40)]), (4, 2, 128, 16, [(50, 90), (1, 40)])], ids=["few", "many"])
@pytest.mark.parametrize("form", ["token_major", "head_gap", "odd_gap", "fused_qkv", "o_over_q", "strided_batch", "unlike_caches", "descending"])
def test_attention_paged_views(gpu, stream, form, shape):
    """Caches with the tokens of a page in front of the heads, rows farther apart (on 16-byte boundaries and not), q a view of
    a fused projection, o in place of q, and tables and lengths that are views themselves."""
    rng = np.random.default_rng(9)
    b = Batch(gpu, rng, "f16", *shape[:4], shape[4], pad=1, token_major=form == "token_major", head_gap={"head_gap": 8, "odd_gap": 3}.get(form, 0))
    want, tol = b.expected(1)
    scale, q, o = b.dh ** -0.5, b.q.host.transpose(1, 0, 2), b.o.host.transpose(1, 0, 2)
    qa, oa, batch = b.q.view(q), b.o.view(o), b.batch_args()
    if form == "fused_qkv":
        wide = np.zeros((b.nt, (b.nh + 2 * b.nkvh) * b.dh), np.float16)
        wide[:, :b.nh * b.dh] = b.q.host.reshape(b.nt, -1)
        fused = Buffer(gpu, wide, "f16")
        qa = fused.view(fused.host[:, :b.nh * b.dh].reshape(b.nt, b.nh, b.dh).transpose(1, 0, 2))
    if form == "o_over_q":
        oa = qa
        want[b.start[-1]:] = decode(b.q.host, "f16")[b.start[-1]:]
    if form == "strided_batch":
        t = Buffer(gpu, np.repeat(np.repeat(b.table.host, 2, 0), 3, 1)[::-1, ::-1])
        st, ln = Buffer(gpu, np.repeat(b.q_start.host, 2)), Buffer(gpu, b.kv_len.host[::-1].astype(np.int32))
        batch = t.view(t.host[::-1, ::-1][::2, ::3]) + st.view(st.host[::2]) + ln.view(ln.host[::-1])
    caches = b.cache_args()
    if form == "unlike_caches":  # v with a page's tokens in front of its heads
        v = Buffer(gpu, b.cache[1].host.swapaxes(1, 2), "f16")
        caches = b.cache[0].view() + v.view(v.host.swapaxes(1, 2))
    if form == "descending":  # pages, heads, tokens, q and o in descending order of addresses
        flipped = [Buffer(gpu, c.host[::-1, ::-1, ::-1], "f16") for c in b.cache]
        caches = flipped[0].view(flipped[0].host[::-1, ::-1, ::-1]) + flipped[1].view(flipped[1].host[::-1, ::-1, ::-1])
        qf, of = Buffer(gpu, b.q.host[::-1], "f16"), Buffer(gpu, b.o.host[:, ::-1], "f16")
        qa, oa = qf.view(qf.host[::-1].transpose(1, 0, 2)), of.view(of.host[:, ::-1].transpose(1, 0, 2))
    run(gpu, stream, ophip.AttentionPagedArgs(*qa, *caches, *oa, *batch, 1, scale))
    if form == "descending":
        return check(decode(of.back(stream)[:, ::-1], "f16"), want, tol)
    got = b.q.back(stream) if form == "o_over_q" else b.o.back(stream)
    check(decode(got, "f16"), want, tol)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
def test_attention_paged_scales(gpu, stream, scale):
    b = Batch(gpu, np.random.default_rng(10), "bf16", 4, 2, 64, 16, [(1, 70), (5, 33)])
    want, tol = b.expected(1, scale)
    check(attend(gpu, stream, b, 1, scale=scale), want, tol)


@pytest.mark.parametrize("lens", [[(1, 50), (1, 300)], [(40, 60), (1, 300)]], ids=["few", "many"])
def test_attention_paged_one_key_outweighs_the_others(gpu, stream, lens):
    """Scores up to hundreds: the running maximum has to carry the sums over."""
    b = Batch(gpu, np.random.default_rng(11), "f16", 4, 1, 128, 16, lens)
    b.q = Buffer(gpu, (b.q.host * np.float16(20)).astype(np.float16), "f16")
    want, tol = b.expected(1)
    check(attend(gpu, stream, b, 1), want, tol)


@pytest.mark.parametrize("tile", ["0", "1", "2"])
@pytest.mark.parametrize("kind,value", [("f16", np.nan), ("bf16", np.inf)])
@pytest.mark.parametrize("dh", [64, 128, 40])
def test_attention_paged_what_is_masked_does_not_matter(gpu, stream, monkeypatch, tile, kind, value, dh):
    """Keys and values that are not finite spoil the rows that see them, wherever the mask ends, and no other."""
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
    b = Batch(gpu, np.random.default_rng(19), kind, 4, 2, dh, 16, [(40, 90), (3, 70), (1, 130), (300, 300), (5, 3)])
    bits = lambda x: encode(np.array([x]), kind)[0]

    def put(which, s, key, head, col):
        b.cache_views[which][b.table.host[s, key // 16], head, key % 16, col] = bits(value)

    put(1, 0, 75, 0, 3), put(1, 0, 89, 1, 5), put(1, 1, 69, 0, 0), put(1, 1, 68, 1, dh - 1)
    put(1, 2, 129, 0, 7), put(1, 3, 130, 1, 8), put(1, 3, 200, 0, 1), put(1, 3, 250, 0, 2), put(0, 3, 290, 1, 4), put(1, 4, 1, 0, 6)
    b.cache = [Buffer(gpu, c.host, kind) for c in b.cache]
    b.cache_views = [c.host for c in b.cache]
    for mask in (1, 0):
        gpu.upload(b.o.mem, b.o.host)
        with np.errstate(invalid="ignore"):
            want, tol = b.expected(mask)
        assert not np.isfinite(want).all() and np.isfinite(want).any()
        check(attend(gpu, stream, b, mask), want, tol, "mask %d" % mask)


@pytest.mark.parametrize("lens", [[(1, 50), (1, 300), (1, 9)], [(40, 60), (1, 300), (20, 20)]], ids=["few", "many"])
@pytest.mark.parametrize("dh", [64, 40])
def test_attention_paged_bad_descriptions_stay_inside(gpu, stream, lens, dh):
    """Page numbers that are none of the cache's, lengths beyond the table, token numbers beyond the batch or in descending
    order: no access outside the operands, and the sequences whose description is right get their rows."""
    b = Batch(gpu, np.random.default_rng(12), "f16", 4, 2, dh, 16, lens, junk=0.0)
    want, tol = b.expected(1)
    table = b.table.host.copy()
    table[0] = 0x7FFFFFF0
    b.table = Buffer(gpu, table)
    got = attend(gpu, stream, b, 1)
    first = b.start[1]
    check(got[first:], want[first:], tol[first:])
    for start, length in (([0, 1, 2, 0xFFFFFFFF], [50, 0xFFFFFFFF, 9]), ([5, 3, 1, 0], [50, 300, 9]), ([0, 0xFFFFFFF0, 0, 0xFFFFFFFF], [1, 1, 1])):
        b.q_start, b.kv_len = Buffer(gpu, np.array(start, np.uint32)), Buffer(gpu, np.array(length, np.uint32))
        attend(gpu, stream, b, 1)


@pytest.mark.parametrize("new", [1, 12])
def test_attention_paged_recorded_and_replayed_with_other_lengths(gpu, stream, new):
    """One recorded launch serves growing sequences: lengths and table change on the device between replays."""
    rng = np.random.default_rng(13)
    lens = [(new, 900), (new, 310), (new, 450)]
    b = Batch(gpu, rng, "f16", 8, 2, 128, 32, lens)
    op, args = ophip.AttentionPaged(gpu), b.args(1)
    ws = gpu.malloc(max(16, op.scheme(args, 1 << 40)))
    own = gpu.stream()
    op.launch(args, ws, own)
    own.synchronize()
    own.begin_capture()
    op.launch(args, ws, own)
    graph = own.end_capture()
    for step in range(4):
        b.lens = [(new, l - 53 * step) for _, l in lens]
        gpu.upload(b.kv_len.mem, np.array([l for _, l in b.lens], np.uint32))
        graph.launch(own)
        own.synchronize()
        want, tol = b.expected(1)
        check(decode(b.o.back(own), "f16"), want, tol, "replay %d" % step)
    graph.destroy()
    own.destroy()


def test_attention_paged_offsets_past_32_bits(gpu, stream):
    """Pages 2.5 GiB apart: the cache reaches past 2^32 elements' bytes."""
    dh, nkvh, page, gap, npages = 64, 2, 16, 5 << 29, 3
    mem = [gpu.malloc(gap * (npages - 1) + nkvh * page * dh * 2) for _ in range(2)]
    rng = np.random.default_rng(14)
    rows = [rng.standard_normal((npages, nkvh, page, dh)).astype(np.float16) for _ in range(2)]
    for m, r in zip(mem, rows):
        for i in range(npages):
            gpu.upload(m, r[i], offset=gap * i)
    for lens in ([(1, 48)], [(40, 48)]):
        b = Batch(gpu, rng, "f16", 4, nkvh, dh, page, lens, spare=0)
        cache = TensorLayout(dt.F16, [npages, nkvh, page, dh], [gap, page * dh * 2, dh * 2, 2])
        q, o = b.q.host.transpose(1, 0, 2), b.o.host.transpose(1, 0, 2)
        run(gpu, stream, ophip.AttentionPagedArgs(*b.q.view(q), cache, mem[0], cache, mem[1], *b.o.view(o), *b.batch_args(), 1, 0.125))
        want, tol = b.expected(1, cache=rows)
        check(decode(b.o.back(stream), "f16"), want, tol)


def test_attention_paged_refusals(gpu, stream):
    rng = np.random.default_rng(15)
    b = Batch(gpu, rng, "f16", 4, 2, 64, 16, [(1, 20), (2, 30)])
    op = ophip.AttentionPaged(gpu)

    def refused(kind, at_scheme=True, **change):
        a = b.args(1)
        for k, v in change.items():
            setattr(a, k, v)
        if at_scheme:
            with pytest.raises(ophip.SchemeError) as e:
                op.scheme(a, 1 << 40)
            assert e.value.kind == kind, e.value
        with pytest.raises(ophip.LaunchError) as e:
            op.launch(a, None, stream)
        assert e.value.kind == kind, e.value

    good = b.args(1)
    L = lambda lay, **c: TensorLayout(c.get("dtype", lay.dt), c.get("shape", lay.shape), c.get("strides", lay.strides))
    refused("RankNotSupport", q_layout=TensorLayout(dt.F16, [4, 64], [128, 2]))
    refused("RankNotSupport", k_cache_layout=TensorLayout(dt.F16, [2, 16, 64], [2048, 128, 2]))
    refused("TypeMismatch", v_cache_layout=L(good.v_cache_layout, dtype=dt.BF16))
    refused("TypeNotSupport", page_table_layout=L(good.page_table_layout, dtype=dt.U64))
    refused("TypeNotSupport", kv_len_layout=L(good.kv_len_layout, dtype=dt.F32))
    f64 = {n: L(getattr(good, n), dtype=dt.F64) for n in ("q_layout", "o_layout", "k_cache_layout", "v_cache_layout")}
    refused("TypeNotSupport", **f64)
    refused("ShapeMismatch", o_layout=L(good.o_layout, shape=[4, 3, 32]))
    refused("ShapeMismatch", q_start_layout=L(good.q_start_layout, shape=[2]))
    refused("ShapeMismatch", q_start_layout=L(good.q_start_layout, shape=[0]))
    refused("ShapeMismatch", q_layout=L(good.q_layout, shape=[3, 3, 64]), o_layout=L(good.o_layout, shape=[3, 3, 64]))  # 3 heads over 2
    big = {n: L(getattr(good, n), shape=list(getattr(good, n).shape[:-1]) + [1024]) for n in ("q_layout", "o_layout", "k_cache_layout", "v_cache_layout")}
    refused("ShapeNotSupport", **big)
    refused("ArgsNotSupport", mask=2)
    refused("ArgsNotSupport", at_scheme=False, scale=float("nan"))
    refused("DynamicNotSupport", at_scheme=False, scale=float("inf"))
    refused("StridesNotSupport", at_scheme=False, q_layout=L(good.q_layout, strides=[127, 512, 2]))
    refused("StridesNotSupport", at_scheme=False, kv_len_layout=L(good.kv_len_layout, strides=[6]))
    refused("ShapeNotSupport", at_scheme=False, k_cache_layout=L(good.k_cache_layout, shape=[6, 2, 0, 64]), v_cache_layout=L(good.v_cache_layout, shape=[6, 2, 0, 64]))
    for n in ("q_base", "o_base", "k_cache_base", "v_cache_base", "page_table_base", "q_start_base", "kv_len_base"):
        refused("ArgsNotSupport", at_scheme=False, **{n: None})
    refused("ArgsNotSupport", at_scheme=False, o_base=good.q_base + 64)        # o part over q
    refused("ArgsNotSupport", at_scheme=False, o_base=good.k_cache_base)
    refused("ArgsNotSupport", at_scheme=False, kv_len_base=good.kv_len_base + 2)
    refused("ArgsNotSupport", at_scheme=False, q_base=good.q_base + 1)
    refused("ShapeNotSupport", at_scheme=False, page_table_layout=L(good.page_table_layout, shape=[2, 1 << 28]))  # 2^32 keys
    refused("DynamicNotSupport", at_scheme=False, q_layout=L(good.q_layout, shape=[None, 3, 64]))
    dyn = L(good.q_layout, strides=[None, None, None])
    dyn_args = b.args(1)
    dyn_args.q_layout = dyn
    assert op.scheme(dyn_args, 1 << 40) >= 0
    refused("DynamicNotSupport", at_scheme=False, q_layout=dyn)
    # nothing to do is fine, whatever the bases
    none = b.args(1)
    none.q_layout, none.o_layout = L(good.q_layout, shape=[4, 0, 64]), L(good.o_layout, shape=[4, 0, 64])
    none.q_base = none.o_base = none.k_cache_base = None
    op.launch(none, None, stream)
    # a cache without pages has no keys: every row of a sequence is zero
    bare = b.args(1)
    bare.k_cache_layout, bare.v_cache_layout = (L(good.k_cache_layout, shape=[0, 2, 16, 64]) for _ in range(2))
    run(gpu, stream, bare, op)
    assert (decode(b.o.back(stream), "f16") == 0).all()


# ---- kv_append_paged

def rotated(x, pos, theta):
    """(rope(x), |a| + |b| of each element's pair) in 64 bits; x [t, heads, dh]."""
    if not theta:
        return x, np.zeros_like(x)
    half = x.shape[-1] // 2
    ang = pos.astype(np.float64)[:, None, None] * float(np.float32(theta)) ** (-np.arange(half) / half)
    a, b = x[..., 0::2], x[..., 1::2]
    out, size = np.empty_like(x), np.empty_like(x)
    out[..., 0::2], out[..., 1::2] = a * np.cos(ang) - b * np.sin(ang), a * np.sin(ang) + b * np.cos(ang)
    size[..., 0::2] = size[..., 1::2] = np.abs(a) + np.abs(b)
    return out, size


def append_case(gpu, rng, kind, nkvh, dh, page, lens, pad, pos_type=np.uint32, far=100000, **form):
    b = Batch(gpu, rng, kind, nkvh, nkvh, dh, page, lens, pad=pad, junk=0.25, **form)
    b.k, b.v = (Buffer(gpu, encode(rng.standard_normal((b.nt, nkvh, dh)), kind), kind) for _ in range(2))
    b.pos = Buffer(gpu, rng.integers(0, far, b.nt).astype(pos_type))
    return b


def append_args(b, theta):
    return ophip.KvAppendPagedArgs(*b.k.view(b.k.host.transpose(1, 0, 2)), *b.v.view(b.v.host.transpose(1, 0, 2)), *b.pos.view(), *b.cache_args(), *b.batch_args(), theta)


def check_append(gpu, stream, b, theta, args=None):
    """Runs it and checks the caches: the written rows, and every other bit as it was."""
    run(gpu, stream, args or append_args(b, theta), ophip.KvAppendPaged(gpu))
    new_k, size = rotated(decode(b.k.host, b.kind), b.pos.host, theta)
    got = [c.back(stream) for c in b.cache]
    left = [c.host.copy() for c in b.cache]
    views = lambda arrays: [np.lib.stride_tricks.as_strided(a, v.shape, v.strides) for a, v in zip(arrays, b.cache_views)]
    gv, lv = views(got), views(left)
    for s, (n, l) in enumerate(b.lens):
        for i in range(max(0, n - l), n):
            t, j = b.start[s] + i, l - n + i
            place = (b.table.host[s, j // b.page], slice(None), j % b.page)
            if theta:
                w = new_k[t]
                check(decode(gv[0][place], b.kind), w, HALF[b.kind] * np.abs(w) + 2.0 ** -20 * size[t] + 2.0 ** -25, "k of token %d" % t)
            else:
                assert np.array_equal(gv[0][place].view(np.uint8), b.k.host[t].view(np.uint8))
            assert np.array_equal(gv[1][place].view(np.uint8), b.v.host[t].view(np.uint8))
            for g, o in zip(gv, lv):
                o[place] = g[place]
    for g, o in zip(got, left):
        assert np.array_equal(g.view(np.uint8), o.view(np.uint8))
    return gv


APPENDS = [(1, 64, 16, [(1, 1)]), (2, 128, 7, [(1, 5), (1, 0), (3, 30)]), (8, 128, 16, [(1, 400), (1, 17)]), (4, 64, 32, [(40, 40), (0, 9), (7, 3)]),
           (3, 24, 5, [(6, 11)]), (2, 512, 4, [(3, 9)]), (2, 6, 4, [(3, 9)]), (32, 128, 64, [(9, 70)])]


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("theta", [10000.0, 0.0])
@pytest.mark.parametrize("shape", APPENDS, ids=str)
def test_kv_append_paged(gpu, stream, shape, theta, kind):
    check_append(gpu, stream, append_case(gpu, np.random.default_rng(20), kind, *shape, pad=2), theta)


def test_kv_append_paged_more_than_the_caches_hold(gpu, stream):
    """48 MiB of rows: non-temporal stores."""
    check_append(gpu, stream, append_case(gpu, np.random.default_rng(26), "bf16", 32, 128, 64, [(1000, 1003), (2000, 2000)], 5), 10000.0)


@pytest.mark.parametrize("form", ["token_major", "head_gap", "odd_gap"])
def test_kv_append_paged_views(gpu, stream, form):
    b = append_case(gpu, np.random.default_rng(21), "bf16", 2, 64, 16, [(3, 20), (1, 40)], 1, token_major=form == "token_major",
                    head_gap={"head_gap": 8, "odd_gap": 3}.get(form, 0))
    check_append(gpu, stream, b, 500000.0)


@pytest.mark.parametrize("pos_type,far", [(np.uint32, 1 << 32), (np.int32, 1 << 31), (np.uint64, 1 << 40), (np.int64, 1 << 20)])
def test_kv_append_paged_far_positions(gpu, stream, pos_type, far):
    """Angles of 10^9 radians and more: taken in f64 on both sides (up to 2^40 positions the f64 angle itself is good to 2^-15
    turns, so positions there are whole multiples of a power of two whose low bits carry nothing)."""
    b = append_case(gpu, np.random.default_rng(22), "f32", 2, 64, 16, [(30, 40)], 0, pos_type=pos_type, far=min(far, 1 << 20))
    check_append(gpu, stream, b, 10000.0)
    if far > 1 << 20:  # positions that turn the first pair by whole f64 steps only: the result is a rotation still
        pos = (b.pos.host.astype(np.uint64) * np.uint64(far >> 20)).astype(pos_type)
        b.pos = Buffer(gpu, pos)
        run(gpu, stream, append_args(b, 10000.0), ophip.KvAppendPaged(gpu))
        got = np.array([decode(b.cache[0].back(stream)[b.table.host[0, j // 16], :, j % 16], "f32") for j in range(10, 40)])
        k = decode(b.k.host, "f32")
        norm = lambda x: x[..., 0::2] ** 2 + x[..., 1::2] ** 2
        assert np.allclose(norm(got), norm(k), rtol=2.0 ** -18, atol=0)


def test_kv_append_paged_bad_descriptions_stay_inside(gpu, stream):
    b = append_case(gpu, np.random.default_rng(23), "f16", 2, 64, 16, [(2, 50), (1, 300), (3, 9)], 1)
    table = b.table.host.copy()
    table[0] = 0x7FFFFFF0
    b.table = Buffer(gpu, table)
    run(gpu, stream, append_args(b, 10000.0), ophip.KvAppendPaged(gpu))
    now = [c.back(stream) for c in b.cache]
    assert (now[1] != b.cache[1].host).any(axis=(1, 3)).sum() == 4  # the four tokens of the other two sequences
    for start, length in (([0, 1, 2, 0xFFFFFFFF], [50, 0xFFFFFFFF, 9]), ([5, 3, 1, 0], [50, 300, 9]), ([0, 0xFFFFFFF0, 0, 0xFFFFFFFF], [1, 1, 1])):
        b.q_start, b.kv_len = Buffer(gpu, np.array(start, np.uint32)), Buffer(gpu, np.array(length, np.uint32))
        run(gpu, stream, append_args(b, 10000.0), ophip.KvAppendPaged(gpu))


def test_kv_append_paged_refusals(gpu, stream):
    b = append_case(gpu, np.random.default_rng(24), "f16", 2, 64, 16, [(2, 20)], 0)
    op = ophip.KvAppendPaged(gpu)

    def refused(kind, theta=10000.0, **change):
        a = append_args(b, theta)
        for k, v in change.items():
            setattr(a, k, v)
        with pytest.raises(ophip.LaunchError) as e:
            op.launch(a, None, stream)
        assert e.value.kind == kind, e.value

    good = append_args(b, 10000.0)
    refused("ArgsNotSupport", theta=-1.0)
    refused("ArgsNotSupport", theta=float("nan"))
    refused("DynamicNotSupport", theta=float("inf"))
    refused("ArgsNotSupport", p_base=None)
    refused("TypeNotSupport", p_layout=TensorLayout(dt.F32, [2], [4]))
    refused("ShapeMismatch", p_layout=TensorLayout(dt.U32, [3], [4]))
    refused("ShapeMismatch", k_layout=TensorLayout(dt.F16, [1, 2, 64], [128, 256, 2]))
    refused("TypeMismatch", k_layout=TensorLayout(dt.BF16, [2, 2, 64], [128, 256, 2]))
    refused("StridesNotSupport", k_layout=TensorLayout(dt.F16, [2, 2, 64], [129, 256, 2]))
    refused("ArgsNotSupport", k_base=good.k_cache_base)
    for n in ("k_base", "v_base", "k_cache_base", "v_cache_base", "page_table_base", "q_start_base", "kv_len_base"):
        refused("ArgsNotSupport", **{n: None})
    odd = append_case(gpu, np.random.default_rng(25), "f16", 1, 5, 4, [(2, 6)], 0)
    with pytest.raises(ophip.LaunchError) as e:
        op.launch(append_args(odd, 10000.0), None, stream)
    assert e.value.kind == "ShapeNotSupport"
    check_append(gpu, stream, odd, 0.0)  # without rotation any dimension
    still = append_args(b, 0.0)
    still.p_base = None  # ... and no positions
    check_append(gpu, stream, b, 0.0, still)


# ---- qk_norm_rope

def normed(x, w, pos, theta, eps):
    """(y, tolerance without the rounding) in 64 bits"""
    z = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    y, size = rotated(z, pos, theta)
    size = size if theta else np.abs(z)
    return y, size * ((x.shape[-1] / 2 + 8) * E + 2.0 ** -20) + 2.0 ** -25


NORMS = [(1, 4, 1, 64), (3, 32, 8, 128), (5, 7, 0, 128), (2, 0, 3, 64), (9, 3, 2, 96), (4, 2, 2, 256), (3, 2, 1, 512), (2, 3, 1, 2), (3, 2, 2, 20), (70, 5, 1, 8)]


@pytest.mark.parametrize("kind,weight", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("theta", [10000.0, 0.0])
@pytest.mark.parametrize("shape", NORMS, ids=str)
def test_qk_norm_rope(gpu, stream, shape, theta, kind, weight):
    rng = np.random.default_rng(30)
    nt, nh, nkh, dh = shape
    check_norm(gpu, stream, rng, nt, nh, nkh, dh, kind, weight, theta)


def check_norm(gpu, stream, rng, nt, nh, nkh, dh, kind, weight, theta, form="apart", scale=1.5, eps=1e-6):
    fused = np.concatenate([rng.standard_normal((nt, nh * dh)) * scale, rng.standard_normal((nt, nkh * dh)) * scale, rng.standard_normal((nt, 3 if form == "odd" else 8))], 1)
    x = Buffer(gpu, encode(fused, kind), kind)
    parts = [x.host[:, :nh * dh].reshape(nt, nh, dh), x.host[:, nh * dh:(nh + nkh) * dh].reshape(nt, nkh, dh)]
    parts = [np.lib.stride_tricks.as_strided(x.host[:, a:], (nt, h, dh), (x.host.strides[0], dh * x.host.itemsize, x.host.itemsize)) for a, h in ((0, nh), (nh * dh, nkh))]
    w = [Buffer(gpu, encode(1 + 0.2 * rng.standard_normal(dh), weight), weight) for _ in range(2)]
    pos = Buffer(gpu, rng.integers(0, 100000, nt).astype(np.uint32))
    if form == "in_place":
        ys, args_y = [x, x], [x.view(p) for p in parts]
    else:
        ys = [Buffer(gpu, np.zeros((nt, max(h, 1), dh), store(kind)), kind) for h in (nh, nkh)]
        args_y = [y.view(y.host[:, :h]) for y, h in zip(ys, (nh, nkh))]
    run(gpu, stream, ophip.QkNormRopeArgs(*args_y[0], *x.view(parts[0]), *w[0].view(), *args_y[1], *x.view(parts[1]), *w[1].view(), *pos.view(), eps, theta), ophip.QkNormRope(gpu))
    for i, h in enumerate((nh, nkh)):
        got = ys[i].back(stream)
        if form == "in_place":
            got = got[:, (0, nh * dh)[i]:][:, :h * dh].reshape(nt, h, dh)
        else:
            got = got[:, :h]
        y, tol = normed(decode(parts[i], kind), decode(w[i].host, weight), pos.host, theta, float(np.float32(eps)))
        check(decode(got, kind), y, tol + HALF[kind] * np.abs(y), "qk"[i])
    if form == "in_place":
        assert np.array_equal(x.back(stream)[:, (nh + nkh) * dh:], x.host[:, (nh + nkh) * dh:])


@pytest.mark.parametrize("form", ["in_place", "odd"])
@pytest.mark.parametrize("dh", [64, 128, 40])
def test_qk_norm_rope_views(gpu, stream, form, dh):
    """q and k views of one fused projection, in place and not, its rows on 16-byte boundaries and not."""
    check_norm(gpu, stream, np.random.default_rng(31), 6, 4, 2, dh, "f16", "f32", 10000.0, form)


@pytest.mark.parametrize("scale", [0.0, 1e-4, 200.0])
def test_qk_norm_rope_small_and_large_rows(gpu, stream, scale):
    check_norm(gpu, stream, np.random.default_rng(32), 4, 3, 2, 128, "f16", "f16", 10000.0, scale=scale, eps=1e-5)


def test_qk_norm_rope_many_tokens(gpu, stream):
    check_norm(gpu, stream, np.random.default_rng(33), 1500, 4, 1, 64, "bf16", "f32", 10000.0)


@pytest.mark.parametrize("nt,nh,nkh,dh", [(4099, 2, 1, 64), (4096, 0, 1, 512), (4097, 3, 0, 8), (4100, 1, 2, 96), (4101, 32, 8, 128)])
def test_qk_norm_rope_several_tokens_per_workgroup(gpu, stream, nt, nh, nkh, dh):
    """From 4096 tokens on a workgroup takes several, the last one fewer; the largest result goes out in non-temporal stores."""
    check_norm(gpu, stream, np.random.default_rng(34), nt, nh, nkh, dh, "f16", "f16", 10000.0)


def test_qk_norm_rope_refusals(gpu, stream):
    op = ophip.QkNormRope(gpu)
    mem = gpu.malloc(1 << 16)
    lay = lambda h, d=64, t=dt.F16, n=2: TensorLayout.new_contiguous(t, [n, h, d])
    w = lambda d=64, t=dt.F16: TensorLayout.new_contiguous(t, [d])
    p = TensorLayout.new_contiguous(dt.U32, [2])
    base = lambda i: mem.ptr + 4096 * i

    def make(**change):
        a = ophip.QkNormRopeArgs(lay(4), base(0), lay(4), base(1), w(), base(2), lay(2), base(3), lay(2), base(4), w(), base(5), p, base(6), 1e-5, 10000.0)
        for k, v in change.items():
            setattr(a, k, v)
        return a

    op.launch(make(), None, stream)
    stream.synchronize()

    def refused(kind, **change):
        with pytest.raises(ophip.LaunchError) as e:
            op.launch(make(**change), None, stream)
        assert e.value.kind == kind, e.value

    refused("ShapeMismatch", q_layout=lay(3))
    refused("ShapeMismatch", kw_layout=w(32))
    refused("ShapeMismatch", p_layout=TensorLayout.new_contiguous(dt.U32, [3]))
    refused("TypeMismatch", k_layout=lay(2, t=dt.BF16))
    refused("TypeMismatch", kw_layout=w(t=dt.F32))
    refused("TypeNotSupport", qw_layout=w(t=dt.BF16), kw_layout=w(t=dt.BF16))
    refused("TypeNotSupport", p_layout=TensorLayout.new_contiguous(dt.F32, [2]))
    refused("RankNotSupport", q_layout=w())
    odd = {n: lay(h, 63) for n, h in (("qy_layout", 4), ("q_layout", 4), ("ky_layout", 2), ("k_layout", 2))}
    refused("ShapeNotSupport", qw_layout=w(63), kw_layout=w(63), **odd)
    refused("StridesNotSupport", q_layout=TensorLayout(dt.F16, [2, 4, 64], [1024, 256, 4]))
    refused("ArgsNotSupport", qy_base=base(1) + 2)
    refused("ArgsNotSupport", theta=-3.0)
    refused("DynamicNotSupport", epsilon=float("inf"))
    for n in ("qy_base", "q_base", "qw_base", "ky_base", "k_base", "kw_base", "p_base"):
        refused("ArgsNotSupport", **{n: None})
    op.launch(make(p_base=None, theta=0.0), None, stream)
    stream.synchronize()


# ---- together: prompts of two sequences, then decode steps, each step norm + rope, append, attention over the cache

@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_a_prompt_and_decode_steps_over_a_paged_cache(gpu, stream, kind):
    rng = np.random.default_rng(40)
    nh, nkvh, dh, page, theta, eps = 8, 2, 64, 16, 10000.0, 1e-6
    npages, cols = 12, 5
    u = HALF[kind]
    table = Buffer(gpu, rng.permutation(npages)[:2 * cols].reshape(2, cols).astype(np.uint32))
    cache = [Buffer(gpu, encode(np.full((npages, nkvh, page, dh), np.nan), kind), kind) for _ in range(2)]
    w = [Buffer(gpu, encode(1 + 0.2 * rng.standard_normal(dh), "f32"), "f32") for _ in range(2)]
    norm, append, attention = ophip.QkNormRope(gpu), ophip.KvAppendPaged(gpu), ophip.AttentionPaged(gpu)
    past = [[[], []], [[], []]]  # per sequence: its keys and values as the cache holds them, in 64 bits
    length = [0, 0]
    for new in ([37, 20], [1, 1], [1, 1], [1, 0], [5, 30]):
        nt = sum(new)
        length = [l + n for l, n in zip(length, new)]
        start = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        pos = np.concatenate([np.arange(l - n, l) for l, n in zip(length, new)]).astype(np.uint32)
        qkv = Buffer(gpu, encode(rng.standard_normal((nt, (nh + 2 * nkvh) * dh)), kind), kind)
        heads = lambda a, h: np.lib.stride_tricks.as_strided(a[:, 0:], (nt, h, dh), (qkv.host.strides[0], dh * SIZE[kind], SIZE[kind]))
        q, k, v = heads(qkv.host, nh), heads(qkv.host[:, nh * dh:], nkvh), heads(qkv.host[:, (nh + nkvh) * dh:], nkvh)
        o = Buffer(gpu, np.zeros((nt, nh, dh), store(kind)), kind)
        st, ln, ps = Buffer(gpu, start), Buffer(gpu, np.array(length, np.uint32)), Buffer(gpu, pos)
        batch, caches = table.view() + st.view() + ln.view(), cache[0].view() + cache[1].view()
        norm.launch(ophip.QkNormRopeArgs(*qkv.view(q), *qkv.view(q), *w[0].view(), *qkv.view(k), *qkv.view(k), *w[1].view(), *ps.view(), eps, theta), None, stream)
        append.launch(ophip.KvAppendPagedArgs(*qkv.view(k.transpose(1, 0, 2)), *qkv.view(v.transpose(1, 0, 2)), *ps.view(), *caches, *batch, 0.0), None, stream)
        attention.launch(ophip.AttentionPagedArgs(*qkv.view(q.transpose(1, 0, 2)), *caches, *o.view(o.host.transpose(1, 0, 2)), *batch, 1, dh ** -0.5), None, stream)
        stream.synchronize()
        got_o, got_qkv = decode(o.back(stream), kind), qkv.back(stream)
        # each step's inputs to the next are checked, and taken as they came out
        for i, (a, h) in enumerate(((0, nh), (nh * dh, nkvh))):
            y, tol = normed(decode(heads(qkv.host[:, a:], h), kind), decode(w[i].host, "f32"), pos, theta, eps)
            check(decode(heads(got_qkv[:, a:], h), kind), y, tol + u * np.abs(y))
        qn, kn, vn = decode(heads(got_qkv, nh), kind), decode(heads(got_qkv[:, nh * dh:], nkvh), kind), decode(v, kind)
        for s in range(2):
            for t in range(start[s], start[s + 1]):
                past[s][0].append(kn[t])
                past[s][1].append(vn[t])
                keys, values = np.array(past[s][0]), np.array(past[s][1])
                for h in range(nh):
                    kk, vv = keys[:, h // 4], values[:, h // 4]
                    x = kk @ qn[t, h] * dh ** -0.5
                    pr = np.exp(x - x.max())
                    pr /= pr.sum()
                    big = (np.abs(kk) @ np.abs(qn[t, h])).max() * dh ** -0.5
                    check(got_o[t, h], pr @ vv, (2 * u + 2 * (dh + 8) * E * big + 2.0 ** -20) * (pr @ np.abs(vv)) + 2.0 ** -25, "token %d head %d" % (t, h))


def test_two_streams_share_the_operators(gpu):
    """One operator on two streams with a workspace each: neither sees the other's partial results."""
    rng = np.random.default_rng(41)
    op = ophip.AttentionPaged(gpu)
    jobs = []
    for lens in ([(1, 2000)], [(1, 1500), (1, 900)]):
        b = Batch(gpu, rng, "f16", 4, 1, 64, 16, lens)
        args, s = b.args(1), gpu.stream()
        jobs.append((b, args, s, gpu.malloc(max(16, op.scheme(args, 1 << 40)))))
    for _ in range(3):
        for b, args, s, ws in jobs:
            op.launch(args, ws, s)
    for b, args, s, ws in jobs:
        want, tol = b.expected(1)
        check(decode(b.o.back(s), "f16"), want, tol)
        s.destroy()


def test_a_stream_made_elsewhere(gpu):
    """ExternalStream takes a hipStream_t it did not make: the operators run on it."""
    own = gpu.stream()
    s = ophip.ExternalStream(gpu, own.handle.value)
    b = Batch(gpu, np.random.default_rng(42), "f16", 2, 1, 64, 16, [(1, 40)])
    ophip.AttentionPaged(gpu).launch(b.args(1), None, s)
    own.synchronize()
    want, tol = b.expected(1)
    check(decode(b.o.back(own), "f16"), want, tol)
    own.destroy()


def test_null_operators_and_arguments(gpu):
    L = ophip.lib()
    ws = ctypes.c_size_t(0)
    for n in ("attention_paged", "kv_append_paged", "qk_norm_rope"):
        assert getattr(L, "ophip_%s_create" % n)(None, None) == 8
        assert getattr(L, "ophip_%s_launch" % n)(None, None, None, ctypes.c_size_t(0), None) == 8
        assert getattr(L, "ophip_%s_scheme" % n)(None, None, ctypes.c_size_t(0), ctypes.byref(ws)) == 8
        getattr(L, "ophip_%s_destroy" % n)(None)


# ---- what the choice of tile by size would leave out: each batch on the tiles that others of its kind have

TILED = [s for s in SHAPES if s[2] in (64, 128)]


@pytest.mark.parametrize("tile", ["0", "1", "2"])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("shape", TILED, ids=lambda s: "%d-%d-%d-%d-%s" % (s[0], s[1], s[2], s[3], "_".join("%dof%d" % x for x in s[4])))
def test_attention_paged_shapes_on_every_tile(gpu, stream, monkeypatch, shape, kind, tile):
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
    test_attention_paged(gpu, stream, shape, 1, kind)


@pytest.mark.parametrize("tile", ["0", "1", "2"])
@pytest.mark.parametrize("form", ["token_major", "head_gap", "odd_gap", "fused_qkv", "o_over_q", "strided_batch", "unlike_caches", "descending"])
@pytest.mark.parametrize("dh", [64, 128])
def test_attention_paged_views_on_every_tile(gpu, stream, monkeypatch, form, dh, tile):
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
    test_attention_paged_views(gpu, stream, form, (4, 2, dh, 16, [(50, 90), (1, 40), (3, 3)]))


@pytest.mark.parametrize("tile", ["1", "2"])
def test_attention_paged_hard_batches_on_large_tiles(gpu, stream, monkeypatch, tile):
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
    test_attention_paged_one_key_outweighs_the_others(gpu, stream, [(40, 60), (1, 300)])
    test_attention_paged_offsets_past_32_bits(gpu, stream)
    test_attention_paged_recorded_and_replayed_with_other_lengths(gpu, stream, 12)
    for lens in ([(1, 50), (1, 300), (1, 9)], [(40, 60), (1, 300), (20, 20)]):
        test_attention_paged_bad_descriptions_stay_inside(gpu, stream, lens, 64)


@pytest.mark.parametrize("tile", ["0", "1"])
@pytest.mark.parametrize("count", [65, 600])
def test_attention_paged_many_sequences_on_every_tile(gpu, stream, monkeypatch, count, tile):
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
    test_attention_paged_many_sequences(gpu, stream, count, 2)


@pytest.mark.parametrize("lens,nh,nkvh", [([(600, 600), (3, 900)], 4, 4), ([(2, 700)] * 5 + [(40, 300)], 16, 2), ([(1, 260)] * 40, 16, 8), ([(1200, 1200)], 8, 1)],
                         ids=["prompt", "chunks", "decode", "long"])
@pytest.mark.parametrize("dh", [64, 128])
def test_attention_paged_sizes_between_the_kernels(gpu, stream, lens, nh, nkvh, dh):
    """On the tiles that the sizes choose, with ranges cut for one workgroup per CU and for more."""
    b = Batch(gpu, np.random.default_rng(41), "bf16", nh, nkvh, dh, 16, lens, pad=2)
    want, tol = b.expected(1)
    check(attend(gpu, stream, b, 1), want, tol)


@pytest.mark.parametrize("nt,nh,nkh,dh", [(255, 2, 1, 64), (256, 2, 1, 64), (257, 4, 4, 128), (511, 6, 2, 128), (513, 6, 2, 128), (1029, 17, 3, 64), (2049, 5, 2, 128),
                                          (2051, 1, 0, 8), (300, 0, 3, 512), (600, 65, 1, 96)])
def test_qk_norm_rope_two_four_and_eight_tokens_per_workgroup(gpu, stream, nt, nh, nkh, dh):
    check_norm(gpu, stream, np.random.default_rng(42), nt, nh, nkh, dh, "f16", "f32", 10000.0)
    check_norm(gpu, stream, np.random.default_rng(43), nt, nh, nkh, dh, "bf16", "bf16", 0.0)


@pytest.mark.parametrize("tile", ["0", "1"])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dh", [8, 24, 56, 72, 80, 96, 120, 136, 192, 256])
def test_attention_paged_head_dimensions_between(gpu, stream, monkeypatch, dh, kind, tile):
    """Multiples of 8 that the matrix kernels fill up with zeros; NaN next to every row of the caches."""
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
    for mask in (1, 0):
        b = Batch(gpu, np.random.default_rng(44), kind, 4, 2, dh, 24, [(40, 90), (1, 600), (9, 9), (3, 2), (130, 200)], pad=1, head_gap=8)
        want, tol = b.expected(mask)
        check(attend(gpu, stream, b, mask), want, tol)


@pytest.mark.parametrize("tile", ["0", "1"])
@pytest.mark.parametrize("form", ["token_major", "odd_gap", "fused_qkv", "o_over_q", "unlike_caches", "descending"])
@pytest.mark.parametrize("dh", [40, 96, 256])
def test_attention_paged_views_of_other_head_dimensions(gpu, stream, monkeypatch, form, dh, tile):
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
    test_attention_paged_views(gpu, stream, form, (4, 2, dh, 16, [(50, 90), (1, 40), (3, 3)]))


@pytest.mark.parametrize("tile", ["0", "1"])
@pytest.mark.parametrize("kind,value", [("f16", np.nan), ("bf16", np.inf)])
@pytest.mark.parametrize("dh", [96, 200])
def test_attention_paged_what_is_masked_does_not_matter_for_other_heads(gpu, stream, monkeypatch, tile, kind, value, dh):
    test_attention_paged_what_is_masked_does_not_matter(gpu, stream, monkeypatch, tile, kind, value, dh)


@pytest.mark.parametrize("dh", [36, 100, 250, 264, 512])
def test_attention_paged_head_dimensions_of_no_matrix_kernel(gpu, stream, dh):
    for kind in ("f16", "bf16", "f32"):
        b = Batch(gpu, np.random.default_rng(45), kind, 4, 2, dh, 24, [(7, 90), (1, 200), (9, 9), (3, 2)], pad=1, head_gap=4)
        want, tol = b.expected(1)
        check(attend(gpu, stream, b, 1), want, tol)


@pytest.mark.parametrize("kind,dh", [("f32", 64), ("f32", 100), ("f32", 250), ("f32", 512), ("bf16", 36), ("f16", 500)])
def test_attention_paged_more_rows_of_no_matrix_kernel(gpu, stream, kind, dh):
    """Beyond two rows to a CU, each has four waves."""
    for mask in (1, 0):
        b = Batch(gpu, np.random.default_rng(46), kind, 8, 2, dh, 7, [(80, 95), (1, 40), (3, 2)], pad=2, head_gap=4)
        want, tol = b.expected(mask)
        check(attend(gpu, stream, b, mask), want, tol)


@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_attention_paged_what_is_masked_does_not_matter_in_f32(gpu, stream, monkeypatch, value):
    test_attention_paged_what_is_masked_does_not_matter(gpu, stream, monkeypatch, "0", "f32", value, 100)


@pytest.mark.parametrize("tile,dh", [("0", 64), ("0", 96), ("1", 128), ("1", 200), ("2", 128)])
@pytest.mark.parametrize("form", ["token_major", "fused_qkv", "o_over_q", "strided_batch", "descending"])
def test_attention_paged_views_of_long_caches(gpu, stream, monkeypatch, form, tile, dh):
    """Lengths at which ranges are cut, so that the join writes o."""
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
    test_attention_paged_views(gpu, stream, form, (4, 2, dh, 32, [(20, 1500), (1, 2100), (3, 3), (5, 1200)]))


@pytest.mark.parametrize("tile", ["0", "1", "2"])
def test_attention_paged_tokens_in_front_of_the_first_sequence(gpu, stream, monkeypatch, tile):
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
    b = Batch(gpu, np.random.default_rng(47), "f16", 4, 2, 128, 16, [(30, 70), (1, 1400), (40, 55)], pad=3)
    b.lens[0], b.start[0] = (23, 70), 7  # seven tokens of no sequence, then the first's 23
    b.q_start = Buffer(gpu, b.start)
    want, tol = b.expected(1)
    check(attend(gpu, stream, b, 1), want, tol)


@pytest.mark.parametrize("nh,nkvh", [(128, 1), (96, 2), (64, 64), (130, 2)])
def test_attention_paged_wide_groups_and_many_heads(gpu, stream, nh, nkvh):
    b = Batch(gpu, np.random.default_rng(48), "bf16", nh, nkvh, 64, 16, [(1, 90), (2, 33), (3, 3)], pad=1)
    want, tol = b.expected(1)
    check(attend(gpu, stream, b, 1), want, tol)


@pytest.mark.parametrize("nt,nh,nkh,dh", [(600, 6, 2, 128), (300, 2, 2, 64), (2100, 3, 1, 64)])
def test_qk_norm_rope_in_place_with_several_tokens_per_workgroup(gpu, stream, nt, nh, nkh, dh):
    check_norm(gpu, stream, np.random.default_rng(49), nt, nh, nkh, dh, "f16", "f32", 10000.0, "in_place")


# ---- tiles of 128 rows whose keys two groups of waves take in turn

@pytest.mark.parametrize("mask", [1, 0])
@pytest.mark.parametrize("lens", [[(1, 700), (3, 9), (0, 5)], [(300, 330)], [(17, 400), (1, 1500), (40, 40)], [(1100, 1100)], [(5, 2)] + [(1, 30)] * 66 + [(30, 600)],
                                  [(20, 64), (20, 65), (20, 128), (20, 129), (33, 33), (20, 192)]],
                         ids=["decode", "prompt", "mixed", "long", "many", "edges"])
@pytest.mark.parametrize("dh", [64, 128])
def test_attention_paged_in_two_groups(gpu, stream, monkeypatch, lens, mask, dh):
    test_attention_paged_every_size_of_tile(gpu, stream, monkeypatch, "3", lens, mask, dh)


@pytest.mark.parametrize("form", ["token_major", "head_gap", "fused_qkv", "o_over_q", "strided_batch", "unlike_caches", "descending"])
@pytest.mark.parametrize("dh", [64, 128])
def test_attention_paged_views_in_two_groups(gpu, stream, monkeypatch, form, dh):
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", "3")
    test_attention_paged_views(gpu, stream, form, (4, 2, dh, 16, [(50, 290), (1, 40), (3, 3), (20, 1500)]))


@pytest.mark.parametrize("slots", ["1", "3", "40"])
def test_attention_paged_key_ranges_in_two_groups(gpu, stream, monkeypatch, slots):
    test_attention_paged_few_and_many_key_ranges(gpu, stream, monkeypatch, "3", slots)


@pytest.mark.parametrize("kind,value", [("f16", np.nan), ("bf16", np.inf)])
@pytest.mark.parametrize("dh", [64, 128])
def test_attention_paged_what_is_masked_does_not_matter_in_two_groups(gpu, stream, monkeypatch, kind, value, dh):
    test_attention_paged_what_is_masked_does_not_matter(gpu, stream, monkeypatch, "3", kind, value, dh)


def test_attention_paged_hard_batches_in_two_groups(gpu, stream, monkeypatch):
    test_attention_paged_hard_batches_on_large_tiles(gpu, stream, monkeypatch, "3")
    test_attention_paged_many_sequences_on_every_tile(gpu, stream, monkeypatch, 600, "3")


# ---- f32 on the matrix cores

@pytest.mark.parametrize("mask", [1, 0])
@pytest.mark.parametrize("lens", [[(1, 700), (3, 9), (0, 5)], [(300, 330)], [(17, 400), (1, 1500), (40, 40)], [(5, 2)] + [(1, 30)] * 66 + [(30, 600)],
                                  [(20, 32), (20, 33), (16, 64), (15, 65), (33, 33), (1, 0), (8, 96)]],
                         ids=["decode", "prompt", "mixed", "many", "edges"])
@pytest.mark.parametrize("dh", [4, 36, 64, 100, 128, 200, 256])
def test_attention_paged_f32_on_the_matrix_cores(gpu, stream, monkeypatch, lens, mask, dh):
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", "1")
    b = Batch(gpu, np.random.default_rng(50), "f32", 4, 2, dh, 24, lens, pad=1, head_gap=4)
    want, tol = b.expected(mask)
    check(attend(gpu, stream, b, mask), want, tol)


@pytest.mark.parametrize("tile", ["0", "1"])
@pytest.mark.parametrize("dh", [64, 100, 256])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_attention_paged_f32_what_is_masked_does_not_matter(gpu, stream, monkeypatch, tile, dh, value):
    test_attention_paged_what_is_masked_does_not_matter(gpu, stream, monkeypatch, tile, "f32", value, dh)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
@pytest.mark.parametrize("form", ["apart", "o_over_q", "tokens_first"])
def test_attention_paged_f32_scales_and_views(gpu, stream, monkeypatch, scale, form):
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", "1")
    b = Batch(gpu, np.random.default_rng(51), "f32", 6, 2, 96, 16, [(40, 90), (9, 9), (1, 300)], pad=2, token_major=form == "tokens_first")
    want, tol = b.expected(1, scale)
    if form != "o_over_q":
        return check(attend(gpu, stream, b, 1, scale=scale), want, tol)
    q = b.q.view(b.q.host.transpose(1, 0, 2))
    want[b.start[-1]:] = decode(b.q.host, "f32")[b.start[-1]:]
    run(gpu, stream, ophip.AttentionPagedArgs(*q, *b.cache_args(), *q, *b.batch_args(), 1, scale))
    check(decode(b.q.back(stream), "f32"), want, tol)


def test_attention_paged_f32_hard_batches(gpu, stream, monkeypatch):
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", "1")
    b = Batch(gpu, np.random.default_rng(52), "f32", 4, 1, 128, 16, [(40, 60), (1, 300)])
    b.q = Buffer(gpu, b.q.host * np.float32(20), "f32")
    want, tol = b.expected(1)
    check(attend(gpu, stream, b, 1), want, tol)
    b = Batch(gpu, np.random.default_rng(53), "f32", 4, 2, 64, 16, [(40, 60), (1, 300), (20, 20)], junk=0.0)
    for start, length in (([0, 1, 2, 0xFFFFFFFF], [50, 0xFFFFFFFF, 9]), ([5, 3, 1, 0], [50, 300, 9]), ([0, 0xFFFFFFF0, 0, 0xFFFFFFFF], [1, 1, 1])):
        b.table = Buffer(gpu, np.full_like(b.table.host, 0x7FFFFFF0))
        b.q_start, b.kv_len = Buffer(gpu, np.array(start, np.uint32)), Buffer(gpu, np.array(length, np.uint32))
        attend(gpu, stream, b, 1)


# ---- values that are not finite where a row sees them

def with_values(gpu, b, values):
    """The batch with single elements of its caches replaced: (0: k, 1: v; sequence, key, head, column or slice, value)."""
    for which, s, key, head, col, value in values:
        b.cache_views[which][b.table.host[s, key // b.page], head, key % b.page, col] = encode(np.array([value]), b.kind)[0]
    b.cache = [Buffer(gpu, c.host, b.kind) for c in b.cache]
    b.cache_views = [c.host for c in b.cache]
    return b


EVERY_KERNEL = [("f16", 64, "0"), ("f16", 64, "1"), ("bf16", 64, "3"), ("bf16", 128, "0"), ("f16", 128, "1"), ("bf16", 128, "2"), ("f16", 128, "3"), ("f16", 96, "0"),
                ("bf16", 200, "1"), ("bf16", 36, "0"), ("f16", 500, "0"), ("f32", 64, "0"), ("f32", 128, "0"), ("f32", 100, "1"), ("f32", 256, "1")]


@pytest.mark.parametrize("kind,dh,tile", EVERY_KERNEL)
@pytest.mark.parametrize("heads", [2, 40])
def test_attention_paged_a_key_that_is_nan_is_not_dropped(gpu, stream, monkeypatch, kind, dh, tile, heads):
    """NaN in the newest key, which one wave may hold alone, or in the first: every row that sees it is NaN."""
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
    b = Batch(gpu, np.random.default_rng(60), kind, heads, 1, dh, 16, [(1, 9), (1, 17), (1, 65), (1, 129), (1, 1), (2, 33), (1, 40), (20, 81)])
    with_values(gpu, b, [(0, s, l - 1, 0, 0, np.nan) for s, (_, l) in enumerate(b.lens) if s != 6] + [(0, 6, 0, 0, 0, np.nan)])
    for mask in (1, 0):
        gpu.upload(b.o.mem, b.o.host)
        want, tol = b.expected(mask)
        assert np.isnan(want).any(-1).sum() >= 8 * heads
        check(attend(gpu, stream, b, mask), want, tol, "mask %d" % mask)


@pytest.mark.parametrize("kind,dh,tile", EVERY_KERNEL)
@pytest.mark.parametrize("heads", [2, 18])
def test_attention_paged_rows_whose_scores_are_all_minus_infinity(gpu, stream, monkeypatch, kind, dh, tile, heads):
    """A softmax over scores of -inf alone is NaN; zeros are for rows that see no key.  One such key, several, all of a long
    sequence whose keys are cut into ranges, and one that is all but the last; beside them rows that see nothing."""
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
    lens = [(1, 1), (1, 40), (3, 70), (1, 1500), (9, 1100), (5, 3), (30, 20), (1, 90), (1, 0), (9, 1090)]
    b = Batch(gpu, np.random.default_rng(61), kind, heads, 1, dh, 16, lens)
    q = np.abs(decode(b.q.host, kind)) + 0.25
    b.q = Buffer(gpu, encode(q, kind), kind)
    low = [(0, s, j, 0, 0, -np.inf) for s, (_, l) in enumerate(lens) for j in range(l) if s != 9 and not (s == 7 and j == 89)]
    with_values(gpu, b, low)
    for mask in (1, 0):
        gpu.upload(b.o.mem, b.o.host)
        with np.errstate(invalid="ignore"):
            want, tol = b.expected(mask)
        assert np.isnan(want).any() and np.isfinite(want[b.start[9]:]).all()
        assert not mask or (want[b.start[5]:b.start[5] + 2] == 0).all() and np.isnan(want[b.start[5] + 2]).all()
        check(attend(gpu, stream, b, mask), want, tol, "mask %d" % mask)


@pytest.mark.parametrize("kind,dh,tile", EVERY_KERNEL)
@pytest.mark.parametrize("heads", [2, 18])
def test_attention_paged_infinite_values_that_a_row_sees(gpu, stream, monkeypatch, kind, dh, tile, heads):
    """An infinite value makes its column infinite, of its sign, and two of unlike signs NaN; the other columns are as ever."""
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
    b = Batch(gpu, np.random.default_rng(62), kind, heads, 1, dh, 16, [(1, 90), (1, 1), (3, 200), (1, 1500), (9, 150), (1, 300), (30, 140)])
    with_values(gpu, b, [(1, 0, 20, 0, 3, np.inf), (1, 0, 5, 0, 7, -np.inf), (1, 1, 0, 0, 1, np.inf), (1, 2, 40, 0, 0, -np.inf), (1, 2, 100, 0, 0, -np.inf),
                         (1, 3, 700, 0, dh - 1, np.inf), (1, 4, 64, 0, 9, np.inf), (1, 5, 3, 0, 2, np.inf), (1, 5, 130, 0, 2, -np.inf), (1, 6, 10, 0, 12, np.inf)])
    for mask in (1, 0):
        gpu.upload(b.o.mem, b.o.host)
        with np.errstate(invalid="ignore"):
            want, tol = b.expected(mask)
        got = attend(gpu, stream, b, mask)
        off = ~np.isfinite(want)
        assert off.sum() == heads * (2 + 1 + 3 + 1 + 9 + 1 + 30)
        assert np.array_equal(got[off], want[off], equal_nan=True), "mask %d" % mask
        check(got, want, tol, "mask %d" % mask)


# ---- appends to a cache that has no place for them

@pytest.mark.parametrize("dh", [64, 6])
@pytest.mark.parametrize("kv_type,over", [(np.uint32, [17, 40, 0xFFFFFFFF, 18]), (np.int32, [17, 33, -1, 16])])
def test_kv_append_paged_beyond_the_table(gpu, stream, dh, kv_type, over):
    """A sequence that has outgrown its row of the table: tokens whose key has no column are not written, those before them
    are, and no row of the cache that was there changes."""
    b = append_case(gpu, np.random.default_rng(63), "f16", 2, dh, 16, [(1, 16), (4, 16), (2, 16), (4, 16)], 1)
    b.kv_len = Buffer(gpu, np.array(over, kv_type))
    run(gpu, stream, append_args(b, 0.0), ophip.KvAppendPaged(gpu))
    want = [c.host.copy() for c in b.cache]
    for s, (n, _) in enumerate(b.lens):
        for i in range(n):
            key = int(over[s]) - n + i
            if 0 <= key < 16:
                assert s == 3
                for w, x in zip(want, (b.k, b.v)):
                    w[b.table.host[s, 0], :, key] = x.host[b.start[s] + i]
    for c, w in zip(b.cache, want):
        assert np.array_equal(c.back(stream).view(np.uint8), w.view(np.uint8))


def test_kv_append_paged_a_sequence_that_ends_behind_the_batch(gpu, stream):
    """q_start that names more tokens than there are: those that are there are the sequence's first, and get their keys."""
    b = append_case(gpu, np.random.default_rng(64), "bf16", 2, 64, 16, [(3, 20), (2, 30)], 0)
    b.q_start = Buffer(gpu, np.array([0, 3, 9], np.uint32))  # six tokens of the second sequence, two of them here: keys 24, 25
    run(gpu, stream, append_args(b, 0.0), ophip.KvAppendPaged(gpu))
    want = [c.host.copy() for c in b.cache]
    for t, s, key in ((0, 0, 17), (1, 0, 18), (2, 0, 19), (3, 1, 24), (4, 1, 25)):
        for w, x in zip(want, (b.k, b.v)):
            w[b.table.host[s, key // 16], :, key % 16] = x.host[t]
    for c, w in zip(b.cache, want):
        assert np.array_equal(c.back(stream), w)


# ---- results over what other workgroups still read

def test_attention_paged_refuses_results_over_the_description(gpu, stream):
    b = Batch(gpu, np.random.default_rng(65), "f16", 4, 2, 64, 16, [(1, 20), (2, 30)])
    op = ophip.AttentionPaged(gpu)
    for n in ("page_table_base", "q_start_base", "kv_len_base"):
        a = b.args(1)
        setattr(a, n, b.o.mem.ptr + 16)
        with pytest.raises(ophip.LaunchError) as e:
            op.launch(a, None, stream)
        assert e.value.kind == "ArgsNotSupport", n
    op.launch(b.args(1), None, stream)
    stream.synchronize()


def test_kv_append_paged_refuses_caches_over_what_it_reads(gpu, stream):
    b = append_case(gpu, np.random.default_rng(66), "f16", 2, 64, 16, [(1, 20), (2, 30)], 0)
    op = ophip.KvAppendPaged(gpu)
    for which in (0, 1):
        for n in ("page_table_base", "q_start_base", "kv_len_base", "p_base"):
            a = append_args(b, 10000.0)
            setattr(a, n, b.cache[which].mem.ptr + 16)
            with pytest.raises(ophip.LaunchError) as e:
                op.launch(a, None, stream)
            assert e.value.kind == "ArgsNotSupport", n
    a = append_args(b, 10000.0)
    a.v_cache_base = a.k_cache_base  # one cache for both
    with pytest.raises(ophip.LaunchError) as e:
        op.launch(a, None, stream)
    assert e.value.kind == "ArgsNotSupport"
    a = append_args(b, 0.0)
    a.p_base = b.cache[0].mem.ptr  # positions that are not read may lie anywhere
    check_append(gpu, stream, b, 0.0, a)


def test_kv_append_paged_caches_side_by_side_in_one_buffer(gpu, stream):
    """Both caches in one buffer, k's and v's pages in turn: their address ranges meet, their elements do not."""
    b = append_case(gpu, np.random.default_rng(67), "f16", 2, 64, 16, [(1, 20), (2, 30), (7, 7)], 0)
    both = Buffer(gpu, np.stack([c.host for c in b.cache], 1), "f16")
    a = append_args(b, 0.0)
    (a.k_cache_layout, a.k_cache_base), (a.v_cache_layout, a.v_cache_base) = (both.view(both.host[:, i]) for i in (0, 1))
    run(gpu, stream, a, ophip.KvAppendPaged(gpu))
    got = both.back(stream)
    check_append(gpu, stream, b, 0.0)
    for i, c in enumerate(b.cache):
        assert np.array_equal(got[:, i].view(np.uint8), c.back(stream).view(np.uint8))


def test_qk_norm_rope_refuses_results_over_what_it_reads(gpu, stream):
    op, mem = ophip.QkNormRope(gpu), gpu.malloc(1 << 16)
    lay = lambda h: TensorLayout.new_contiguous(dt.F16, [2, h, 64])
    w, p = TensorLayout.new_contiguous(dt.F16, [64]), TensorLayout.new_contiguous(dt.U32, [2])
    base = lambda i: mem.ptr + 4096 * i

    def make(theta=10000.0, **change):
        a = ophip.QkNormRopeArgs(lay(4), base(0), lay(4), base(1), w, base(2), lay(2), base(3), lay(2), base(4), w, base(5), p, base(6), 1e-5, theta)
        for k, v in change.items():
            setattr(a, k, v)
        return a

    for y in (0, 3):
        for n in ("qw_base", "kw_base", "p_base"):
            with pytest.raises(ophip.LaunchError) as e:
                op.launch(make(**{n: base(y) + 16}), None, stream)
            assert e.value.kind == "ArgsNotSupport", n
    for n in ("ky_base", "k_base"):  # the other rows' input or result: the same address
        with pytest.raises(ophip.LaunchError) as e:
            op.launch(make(**{n: base(0)}), None, stream)
        assert e.value.kind == "ArgsNotSupport", n
    with pytest.raises(ophip.LaunchError) as e:
        op.launch(make(q_base=base(3)), None, stream)
    assert e.value.kind == "ArgsNotSupport"
    op.launch(make(theta=0.0, p_base=base(0)), None, stream)
    stream.synchronize()


# ---- which kernel f32 runs on

@pytest.mark.parametrize("nh,nkvh,dh,lens,tiles", [
    (16, 1, 128, [(1, 200)], False),            # one decode step whose 16 rows are a single tile
    (32, 1, 64, [(1, 90), (1, 70)], False),
    (8, 1, 256, [(9, 100)], False),
    (4, 1, 64, [(16, 60)], False),              # 64 rows: one tile, or a workgroup for each
    (12, 4, 64, [(50, 50)], True),              # 600 rows in 12 tiles
    (16, 2, 128, [(49, 50)], False),            # 784 rows: at these sizes a row at a time is still faster
    (40, 1, 128, [(30, 40)], True),
    (16, 2, 200, [(49, 50)], False),
    (20, 1, 256, [(65, 65)], False),
    (20, 1, 256, [(80, 80)], True),
], ids=str)
def test_attention_paged_f32_tiles_only_where_they_fill_the_machine(gpu, stream, monkeypatch, nh, nkvh, dh, lens, tiles):
    """Tiles of 64 rows are never cut into ranges: few of them leave most CUs without work.  The chosen kernel shows in the
    last bits: the two add in different orders."""
    got = {}
    b = Batch(gpu, np.random.default_rng(68), "f32", nh, nkvh, dh, 16, lens)
    for tile in ("0", "1", None):
        monkeypatch.delenv("OPHIP_ATTN_PAGED_TILE", raising=False) if tile is None else monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
        gpu.upload(b.o.mem, b.o.host)
        got[tile] = attend(gpu, stream, b, 1)
    assert not np.array_equal(got["0"], got["1"])
    assert np.array_equal(got[None], got["1" if tiles else "0"])


# ---- what up to 16 rows promise: probabilities that are not rounded to the type

@pytest.mark.parametrize("kind,dh,tile", [("f16", 64, "0"), ("bf16", 64, "1"), ("bf16", 128, "0"), ("f16", 128, "2"), ("bf16", 128, "3"), ("f16", 96, "0"), ("bf16", 256, "1"), ("f16", 8, "0")])
@pytest.mark.parametrize("group", [4, 8])
def test_attention_paged_decode_steps_do_not_round_probabilities(gpu, stream, monkeypatch, kind, dh, tile, group):
    """Values of one sign over a few keys, so that roundings of probabilities do not cancel: within one rounding of the result.
    A probability goes into the product as its rounding and the rounded rest, which leaves u^2 of it (in f16 no less than 2^-32
    of the largest, 2^-27 for up to 32 keys), so the bound is u |o| + (u^2 + 2 (dh + 8) e S + 2^-20) A, with u, e, S and A as above.  Rounded
    probabilities do not stay within it, which is computed here as well."""
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
    rng = np.random.default_rng(70)
    b = Batch(gpu, rng, kind, 2 * group, 2, dh, 16, [(1, int(l)) for l in rng.integers(2, 8, 40)] + [(16 // group, 20)])
    b.cache = [b.cache[0], Buffer(gpu, encode(np.abs(decode(b.cache[1].host, kind)), kind), kind)]
    b.cache_views = [c.host for c in b.cache]
    b.q = Buffer(gpu, encode(decode(b.q.host, kind) * 0.25, kind), kind)  # small scores: what f32 leaves of them is little beside u
    scale, u = float(np.float32(dh ** -0.5)), HALF[kind]
    want, tol = np.zeros((b.nt, b.nh, dh)), np.zeros((b.nt, b.nh, dh))
    q, rounded = decode(b.q.host, kind), np.zeros((b.nt, b.nh, dh))
    for s, (n, l) in enumerate(b.lens):
        k, v = b.keys(s, 0), b.keys(s, 1)
        for i in range(n):
            t, keep = b.start[s] + i, l - n + i + 1
            for h in range(b.nh):
                kk, vv = k[:keep, h // group], v[:keep, h // group]
                x = kk @ q[t, h] * scale
                p = np.exp(x - x.max())
                big = (np.abs(kk) @ np.abs(q[t, h])).max() * scale
                want[t, h] = p @ vv / p.sum()
                tol[t, h] = u * np.abs(want[t, h]) + (u * u + 2 * (dh + 8) * E * big + 2.0 ** -20) * (p @ np.abs(vv) / p.sum()) + 2.0 ** -25
                rounded[t, h] = decode(encode(decode(encode(p, kind), kind) @ vv / p.sum(), kind), kind)
    assert (np.abs(rounded - want) > tol).sum() > 20
    check(attend(gpu, stream, b, 1), want, tol)


# ---- positions beyond 31 and 32 bits

FAR = [(np.uint32, [0, 1, 0x7FFFFFFF, 0x80000000, 0xFFFFFFFF, 3000000019]), (np.int32, [0x7FFFFFFF, 2000000011]),
       (np.uint64, [5, 1 << 32, (1 << 32) + 1, (1 << 33) + 12345, (1 << 40) - 1]), (np.int64, [7, (1 << 32) - 1, (1 << 35) + 977, 3 << 38])]


def rotated_far(x, pos, theta):
    """`rotated` with the angles in 80 bits, and what an angle computed in f64 may be off by: the exponent a of theta^(-k / half) = 2^-a
    and its power are good to (a + 3) 2^-51 relative, rounding by rounding, and (a + 3) 2^-a <= 3: 3 pos 2^-51 radians."""
    assert np.finfo(np.longdouble).nmant >= 63
    half = x.shape[-1] // 2
    freq = np.longdouble(np.float32(theta)) ** (-np.arange(half).astype(np.longdouble) / half)
    ang = np.array([np.longdouble(int(p)) for p in pos])[:, None, None] * freq
    c, s = np.cos(ang).astype(np.float64), np.sin(ang).astype(np.float64)
    a, b = x[..., 0::2], x[..., 1::2]
    out, size = np.empty_like(x), np.empty_like(x)
    out[..., 0::2], out[..., 1::2] = a * c - b * s, a * s + b * c
    size[..., 0::2] = size[..., 1::2] = np.abs(a) + np.abs(b)
    return out, size * (2.0 ** -20 + 3 * 2.0 ** -51 * np.asarray(pos, np.float64)[:, None, None])


@pytest.mark.parametrize("pos_type,far", FAR, ids=lambda x: np.dtype(x).name if isinstance(x, type) else "")
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dh", [64, 6])
@pytest.mark.parametrize("theta", [10000.0, 500000.0])
def test_kv_append_paged_angles_of_far_positions(gpu, stream, pos_type, far, kind, dh, theta):
    n = len(far)
    b = append_case(gpu, np.random.default_rng(71), kind, 2, dh, 16, [(n, n + 13)], 0)
    b.pos = Buffer(gpu, np.array(far, pos_type))
    run(gpu, stream, append_args(b, theta), ophip.KvAppendPaged(gpu))
    want, tol = rotated_far(decode(b.k.host, kind), far, theta)
    back = b.cache[0].back(stream)
    got = np.array([decode(back[b.table.host[0, j // 16], :, j % 16], kind) for j in range(13, 13 + n)])
    check(got, want, tol + HALF[kind] * np.abs(want) + 2.0 ** -25)


@pytest.mark.parametrize("pos_type,far", FAR, ids=lambda x: np.dtype(x).name if isinstance(x, type) else "")
@pytest.mark.parametrize("dh,many", [(64, 1), (6, 1), (128, 300)])
def test_qk_norm_rope_angles_of_far_positions(gpu, stream, pos_type, far, dh, many):
    """Rows of norm 1 before the rotation up to what the norm's own roundings leave; one token per workgroup and several."""
    rng, theta = np.random.default_rng(72), 10000.0
    far = (far * many)[:max(len(far), many)]
    q, k = (Buffer(gpu, encode(rng.standard_normal((len(far), h, dh)), "f32"), "f32") for h in (3, 2))
    qy, ky = (Buffer(gpu, np.zeros(x.host.shape, np.float32), "f32") for x in (q, k))
    w, pos = Buffer(gpu, encode(1 + 0.2 * rng.standard_normal(dh), "f32"), "f32"), Buffer(gpu, np.array(far, pos_type))
    run(gpu, stream, ophip.QkNormRopeArgs(*qy.view(), *q.view(), *w.view(), *ky.view(), *k.view(), *w.view(), *pos.view(), 1e-6, theta), ophip.QkNormRope(gpu))
    for x, y in ((q, qy), (k, ky)):
        x64 = x.host.astype(np.float64)
        z = x64 / np.sqrt((x64 * x64).mean(-1, keepdims=True) + float(np.float32(1e-6))) * w.host.astype(np.float64)
        want, tol = rotated_far(z, far, theta)
        _, size = rotated(z, np.zeros(len(far)), theta)
        check(y.back(stream).astype(np.float64), want, tol + size * (dh / 2 + 8) * E + HALF["f32"] * np.abs(want) + 2.0 ** -25)


# ---- the plan of more sequences than a workgroup has threads, with key ranges

@pytest.mark.parametrize("tile,dh", [("0", 64), ("1", 64), ("2", 128), ("3", 64)])
@pytest.mark.parametrize("count", [65, 300, 1100])
def test_attention_paged_key_ranges_among_many_sequences(gpu, stream, monkeypatch, count, tile, dh):
    """Long sequences at the start, in the middle and at the end of many short ones: the sums that find a workgroup's place carry
    over from round to round, tiles and ranges apart."""
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
    rng = np.random.default_rng(73)
    lens = [(int(n), int(l)) for n, l in zip(rng.integers(0, 3, count), rng.integers(0, 40, count))]
    for s, n, l in ((0, 1, 1700), (1, 20, 1500), (count // 2, 1, 1600), (count // 2 + 1, 40, 1550), (count - 2, 9, 1580), (count - 1, 1, 1900)):
        lens[s] = (n, l)
    b = Batch(gpu, rng, "f16", 2, 1, dh, 32, lens, pad=2)
    op = ophip.AttentionPaged(gpu)
    assert op.scheme(b.args(1), 1 << 40) > 0
    want, tol = b.expected(1)
    check(attend(gpu, stream, b, 1, op=op), want, tol)


@pytest.mark.parametrize("slots", ["1", "3", "40"])
def test_attention_paged_few_and_many_key_ranges_of_256_rows(gpu, stream, monkeypatch, slots):
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", "2")
    monkeypatch.setenv("OPHIP_ATTN_PAGED_SLOTS", slots)
    b = Batch(gpu, np.random.default_rng(74), "bf16", 4, 2, 128, 16, [(20, 2000), (1, 3000), (150, 900)])
    want, tol = b.expected(1)
    check(attend(gpu, stream, b, 1), want, tol)


@pytest.mark.parametrize("dh,tile", [(64, "0"), (64, "1"), (128, "2"), (128, "3"), (96, "0"), (36, "0")])
def test_attention_paged_subnormal_f16_values(gpu, stream, monkeypatch, dh, tile):
    """Values and results below 2^-14, where f16 has steps of 2^-24: nothing is taken for zero."""
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
    b = Batch(gpu, np.random.default_rng(75), "f16", 4, 2, dh, 16, [(1, 1), (3, 40), (30, 64), (1, 300)])
    small = decode(b.cache[1].host, "f16") * 2.0 ** -17
    b.cache[1] = Buffer(gpu, encode(small, "f16"), "f16")
    b.cache_views = [c.host for c in b.cache]
    want, tol = b.expected(1)
    assert np.abs(want).max() < 2.0 ** -14 and (np.abs(want) > tol).mean() > 0.9
    check(attend(gpu, stream, b, 1), want, tol)


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
def test_a_recorded_step_replayed_while_the_sequences_grow(gpu, kind):
    """Norm and rotation, append and attention in one recorded graph, every replay bit for bit what the same calls give one by one on caches of
    their own; inputs, positions, lengths and the table's entries are uploaded between replays."""
    rng = np.random.default_rng(76)
    nh, nkvh, dh, page, theta = 8, 2, 64, 16, 10000.0
    cols, ns = 96, 3  # up to 1536 keys: wide enough for key ranges
    pages = ns * cols
    table = rng.permutation(pages).reshape(ns, cols).astype(np.uint32)
    past = [encode(rng.standard_normal((pages, nkvh, page, dh)), kind) for _ in range(2)]
    w = Buffer(gpu, encode(1 + 0.2 * rng.standard_normal(dh), "f32"), "f32")
    ops = ophip.QkNormRope(gpu), ophip.KvAppendPaged(gpu), ophip.AttentionPaged(gpu)
    sides = []
    for _ in range(2):
        s = {"qkv": Buffer(gpu, np.zeros((ns, (nh + 2 * nkvh) * dh), store(kind)), kind), "cache": [Buffer(gpu, c, kind) for c in past],
             "o": Buffer(gpu, np.zeros((ns, nh, dh), store(kind)), kind), "table": Buffer(gpu, table), "start": Buffer(gpu, np.arange(ns + 1, dtype=np.uint32)),
             "len": Buffer(gpu, np.zeros(ns, np.uint32)), "pos": Buffer(gpu, np.zeros(ns, np.uint32)), "stream": gpu.stream()}
        heads = lambda a, h: np.lib.stride_tricks.as_strided(a, (ns, h, dh), (s["qkv"].host.strides[0], dh * SIZE[kind], SIZE[kind]))
        q, k, v = heads(s["qkv"].host, nh), heads(s["qkv"].host[:, nh * dh:], nkvh), heads(s["qkv"].host[:, (nh + nkvh) * dh:], nkvh)
        at = lambda x: s["qkv"].view(x)
        batch, caches = s["table"].view() + s["start"].view() + s["len"].view(), s["cache"][0].view() + s["cache"][1].view()
        s["args"] = (ophip.QkNormRopeArgs(*at(q), *at(q), *w.view(), *at(k), *at(k), *w.view(), *s["pos"].view(), 1e-6, theta),
                     ophip.KvAppendPagedArgs(*at(k.transpose(1, 0, 2)), *at(v.transpose(1, 0, 2)), *s["pos"].view(), *caches, *batch, 0.0),
                     ophip.AttentionPagedArgs(*at(q.transpose(1, 0, 2)), *caches, *s["o"].view(s["o"].host.transpose(1, 0, 2)), *batch, 1, dh ** -0.5))
        s["ws"] = gpu.malloc(max(16, ops[2].scheme(s["args"][2], 1 << 40)))
        sides.append(s)
    recorded, eager = sides

    def step(s):
        for op, args, ws in zip(ops, s["args"], (None, None, s["ws"])):
            op.launch(args, ws, s["stream"])

    recorded["stream"].begin_capture()
    step(recorded)
    graph = recorded["stream"].end_capture()
    lens = np.array([0, 700, 1500], np.uint32)
    for turn in range(6):
        lens = lens + 1
        x = encode(rng.standard_normal((ns, (nh + 2 * nkvh) * dh)), kind)
        if turn == 3:  # the sequences change places in the batch
            lens, table = lens[::-1].copy(), table[::-1].copy()
        for s in sides:
            for name, value in (("qkv", x), ("len", lens), ("pos", lens - 1), ("table", table)):
                gpu.upload(s[name].mem, np.ascontiguousarray(value))
        graph.launch(recorded["stream"])
        step(eager)
        for s in sides:
            s["stream"].synchronize()
        for name in ("o", "qkv"):
            a, b = (s[name].back(s["stream"]).view(np.uint8) for s in sides)
            assert np.array_equal(a, b), "%s, replay %d" % (name, turn)
        for a, b in zip(recorded["cache"], eager["cache"]):
            assert np.array_equal(a.back(recorded["stream"]).view(np.uint8), b.back(eager["stream"]).view(np.uint8)), turn
        assert np.isfinite(decode(eager["o"].back(eager["stream"]), kind)).all() and (decode(eager["o"].back(eager["stream"]), kind) != 0).any((1, 2)).all()
    graph.destroy()
    for s in sides:
        s["stream"].destroy()


# ---- a row is a mean of values: it does not leave their range

@pytest.mark.parametrize("kind,dh,tile", EVERY_KERNEL)
@pytest.mark.parametrize("value", [1.0, 65504.0, -65504.0])
@pytest.mark.parametrize("spread", [1.0, 4.0])
def test_attention_paged_values_that_are_all_the_same(gpu, stream, monkeypatch, kind, dh, tile, value, spread):
    """Whatever the probabilities, rounded or not: their sum is what they are divided by.  One rounding of the result, the second order of the
    rests (u^2), and the additions of K like-signed terms in f32, each off by e of a sum that is no larger than the last, in the numerator
    and in the sum of probabilities: (u + u^2 + 2 K e) |c|; at the largest value of f16 as well, next to which infinity lies."""
    monkeypatch.setenv("OPHIP_ATTN_PAGED_TILE", tile)
    b = Batch(gpu, np.random.default_rng(77), kind, 4, 2, dh, 16, [(30, 64), (90, 90), (1, 50), (20, 1200), (5, 3), (40, 41)], junk=0.0)
    b.q = Buffer(gpu, encode(decode(b.q.host, kind) * spread, kind), kind)
    c = float(decode(encode(np.array([value]), kind), kind)[0])
    b.cache[1] = Buffer(gpu, encode(np.full(b.cache[1].host.shape, c), kind), kind)
    b.cache_views = [x.host for x in b.cache]
    want = np.full((b.nt, b.nh, dh), c)
    want[b.start[4]:b.start[4] + 2] = 0  # no key
    u = HALF[kind]
    check(attend(gpu, stream, b, 1), want, (u + u * u + 2 * 1200 * E) * np.abs(want))
