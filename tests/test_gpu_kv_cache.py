"""8-bit KV cache and rotary positions on the GPU against the operators in 64 bits (tests/kv_reference.py).

Tolerances, all from the number formats.  u = finfo(io).eps / 2 is the rounding of an output.
* rotary: u |y| + 2^-20 (|x0| + |x1|): cosine and sine are within 2^-22 (two roundings to FP32 and sincospi's 2 ulp), two
  products and a sum of FP32.
* append, evict, read: the stored bytes and scales are exact where the inputs are (no rotary); with rotary an element
  next to a border may land on either side: half a step and what the rotary may be off.
  (An output below the io type's smallest normal number is rounded by half of the fixed step there.)
* attention: scores carry the FP32 sums of exact products: at most d / 16 + 8 additions, each off by at most 2^-22 (the
  tensor pipe truncates) of scale sum |q| |k| =: S, so dS = 2^-22 (d / 16 + 8) S; p is off by 2 dS + 2^-20 (exponential and
  sum) and by 2^-11 of itself in the product with v (f16), so out: u |o| + (2^-11 + 4 dS + 2^-19) sum p |v|,
  lse: dS + 2^-20 (1 + |lse|), weights: (4 dS + 2^-18) w + 2^-22 (sum of what was there).
"""
import math
import random

import pytest
import torch

from tests import kv_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _sl():
    import slora_b200 as sl
    return sl


def _io(name):
    return {"fp16": torch.float16, "bf16": torch.bfloat16}[name]


class World:
    """A cache with random content, garbage in every slot that no sequence owns, and a batch over it."""

    def __init__(self, lens, new, hkv, d, page, kind, seed=0, track=True, spare=2, max_pages=None, n_pages=None, rows_behind=3):
        sl = _sl()
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lens]
        total = n_pages or sum(need) + spare
        order = torch.randperm(total, generator=g)[: sum(need) + spare].tolist()
        width = max_pages or max(1, max(need))
        table = torch.full((len(lens), width), -7, dtype=torch.int64)     # entries behind the last page are not read
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int64)
            at += n
        self.free = order[at:]
        k = torch.randint(0, 256, (total, hkv, page, d), generator=g).to(torch.uint8)     # NaN bytes of e4m3 among them
        v = torch.randint(0, 256, (total, hkv, page, d), generator=g).to(torch.uint8)
        ks, vs = torch.full((total, hkv), math.nan), torch.full((total, hkv), math.nan)
        for i, n in enumerate(lens):
            for b in range(need[i]):
                p, m = int(table[i, b]), min(page, n - b * page)
                for x8, sc in ((k, ks), (v, vs)):
                    x = torch.randn(hkv, m, d, generator=g) * (0.2 + 3 * torch.rand(hkv, 1, 1, generator=g))
                    s = (x.abs().amax((1, 2)) / ref.TOP[kind])
                    y = ref.nearest(x.double() / s[:, None, None].double(), kind).float().to(ref.DTYPE[kind])
                    x8[p, :, :m] = y.view(torch.uint8)
                    sc[p] = s
        self.k8, self.v8 = (x.to(DEV).view(ref.DTYPE[kind]) for x in (k, v))
        self.ks, self.vs = ks.to(DEV), vs.to(DEV)
        self.w = torch.rand(total, hkv, page, generator=g).to(DEV) if track else None
        self.cache = sl.KvCache8.from_buffers([self.k8], [self.v8], [self.ks], [self.vs], [self.w] if track else None)
        self.lens, self.new, self.kind, self.page, self.hkv, self.d = lens, new, kind, page, hkv, d
        # the sequences' rows do not lie in the sequences' order, with gaps between
        starts, at = [0] * len(lens), 1
        for i in reversed(range(len(lens))):
            starts[i] = at
            at += new[i] + (i % 2)
        self.starts, self.T = starts, at + rows_behind
        self.table = table
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        self.batch = sl.KvBatch(table.to(DEV), i32(lens), i32(starts), i32(new), max(new) if new else 0)

    def own_rows(self):
        own = torch.zeros(self.T, dtype=torch.bool)
        for s, n in zip(self.starts, self.new):
            own[s:s + n] = True
        return own.to(DEV)


def _check_attend(w, q, out, lse, weights, w_before, window=0, scale=None):
    d = w.d
    scale = d ** -0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    # below the smallest normal number (2^-14 in fp16) values are a fixed step apart, eps times that number: half of it
    least = torch.finfo(q.dtype).tiny * torch.finfo(q.dtype).eps / 2
    kv, vv = ref.values(w.k8), ref.values(w.v8)
    for i, (n, m, r0) in enumerate(zip(w.lens, w.new, w.starts)):
        if m == 0:
            continue
        k = ref.dense(kv, w.ks.double(), w.table[i], n)
        v = ref.dense(vv, w.vs.double(), w.table[i], n)
        o, z, p, mag, size = ref.attend(k, v, q[r0:r0 + m].double(), window, scale)
        ds = 2.0 ** -22 * (d / 16 + 8) * size
        # f16 holds p vs 32 / ref (ref <= 2 max vs; the largest p is 1 or more): below 2^-14 its steps are 2^-24, so each key
        # may add 2^-25 ref / 32 |v8| <= 2^-29 max |v| where keys of large p have no value
        floor = n * 2.0 ** -29 * float(v.abs().max()) if n else 0.0
        tol = u * o.abs() + (2.0 ** -11 + 4 * ds + 2.0 ** -19) * mag + least + floor
        got = out[r0:r0 + m].double()
        assert torch.isfinite(got).all(), i
        assert bool(((got - o).abs() <= tol).all()), (i, n, m, float(((got - o).abs() / tol).max()))
        if lse is not None:
            y = lse[r0:r0 + m].double()
            none = z == -math.inf
            assert torch.equal(none, y == -math.inf)
            off = (y - z).abs()[~none]
            assert (off <= (ds + 2.0 ** -20 * (1 + z.abs()))[~none]).all(), (i, float(off.max()))
        if weights is not None:
            pages = w.table[i][: -(-n // w.page)].to(DEV)
            have = weights[pages].transpose(0, 1).reshape(w.hkv, -1).double()
            was = w_before[pages].transpose(0, 1).reshape(w.hkv, -1).double()
            off = (have[:, :n] - was[:, :n] - p).abs()
            assert (off <= (4 * ds + 2.0 ** -18) * p + 2.0 ** -22 * (was[:, :n] + p)).all(), (i, float(off.max()))
            assert torch.equal(have[:, n:], was[:, n:])       # slots behind the end are left as they were


def _run_attend(w, hq, io, window=0, scale=None, weights=False, seed=1, q=None):
    g = torch.Generator().manual_seed(seed)
    if q is None:
        q = (torch.randn(w.T, hq, w.d, generator=g) * 1.5).to(_io(io)).to(DEV)
    out = torch.full_like(q, 7.0)
    lse = torch.full((w.T, q.size(1)), 7.0, device=DEV)
    before = None if w.w is None else w.w.clone()
    got = w.cache.attend(0, w.batch, q, out=out, lse=lse, window=window, scale=scale, add_weights=weights)
    torch.cuda.synchronize()
    assert got is out
    _check_attend(w, q, out, lse, w.w if weights else None, before, window, scale)
    rest = ~w.own_rows()
    assert (out[rest] == 7.0).all() and (lse[rest] == 7.0).all()      # rows of no sequence are left as they were
    if not weights and w.w is not None:
        assert torch.equal(w.w, before)
    assert w.batch.status() == 0
    return out, lse


# ---- attention ----------------------------------------------------------------------------------------------------

DECODE = [
    # lens, q heads, KV heads, d, page, kind, io
    ([1], 1, 1, 128, 16, "int8", "fp16"),
    ([1, 2, 15, 16, 17, 63, 64, 65], 2, 2, 128, 16, "int8", "fp16"),
    ([5, 300, 0, 129, 1000], 8, 1, 128, 16, "int8", "bf16"),
    ([31, 64, 700], 8, 2, 64, 32, "e4m3", "fp16"),
    ([31, 64, 700], 12, 4, 256, 64, "int8", "bf16"),
    ([128, 127, 129, 513], 16, 1, 128, 128, "e4m3", "bf16"),
    ([77, 260], 40, 2, 64, 16, "int8", "fp16"),
    ([77, 260], 20, 1, 256, 16, "e4m3", "fp16"),
    ([3000, 10, 9000], 32, 8, 128, 64, "int8", "bf16"),
    ([200 + 37 * i for i in range(33)], 4, 4, 128, 32, "int8", "fp16"),
]


@pytest.mark.parametrize("lens,hq,hkv,d,page,kind,io", DECODE)
def test_decode(lens, hq, hkv, d, page, kind, io):
    w = World(lens, [1] * len(lens), hkv, d, page, kind)
    _run_attend(w, hq, io)
    _run_attend(w, hq, io, weights=True, seed=2)


@pytest.mark.parametrize("window", [1, 16, 50, 64, 500])
def test_decode_window(window):
    w = World([1, 40, 64, 65, 700, 129], [1] * 6, 2, 128, 16, "int8")
    _run_attend(w, 8, "fp16", window=window)
    _run_attend(w, 8, "fp16", window=window, weights=True)


@pytest.mark.parametrize("lens,new,hq,hkv,d,page,kind", [
    ([5, 100, 64, 333], [5, 2, 1, 4], 8, 2, 128, 16, "int8"),
    ([40, 200, 3], [9, 30, 3], 4, 4, 64, 32, "e4m3"),
    ([700, 130], [64, 130], 8, 1, 128, 64, "int8"),
    ([257, 90, 1], [257, 0, 1], 6, 3, 128, 16, "int8"),
    ([100, 60], [33, 60], 2, 1, 256, 16, "e4m3"),
    ([900], [300], 16, 2, 64, 128, "int8"),
    ([2100, 640, 512], [600, 640, 1], 8, 1, 128, 64, "e4m3"),
    ([1500], [1100], 5, 1, 128, 32, "int8"),
])
@pytest.mark.parametrize("window", [0, 70])
def test_several_new_tokens(lens, new, hq, hkv, d, page, kind, window):
    w = World(lens, new, hkv, d, page, kind)
    _run_attend(w, hq, "bf16", window=window)
    _run_attend(w, hq, "fp16", window=window, weights=True)


def test_queries_that_see_nothing():
    # three new tokens over two cached ones: the first query precedes position 0
    w = World([2, 0, 30], [3, 2, 40], 2, 128, 16, "int8")
    out, lse = _run_attend(w, 4, "fp16", weights=True)
    r = w.starts[0]
    assert (out[r] == 0).all() and (lse[r] == -math.inf).all()
    r = w.starts[1]
    assert (out[r:r + 2] == 0).all() and (lse[r:r + 2] == -math.inf).all()
    r = w.starts[2]
    assert (out[r:r + 10] == 0).all() and (lse[r:r + 10] == -math.inf).all() and (lse[r + 10:r + 40] > -100).all()


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 3])
def test_the_widest_window_is_none(window):
    # more new tokens than cached ones: the first queries precede position 0
    w = World([1, 3, 60, 200], [4, 90, 70, 130], 2, 128, 16, "int8")
    q = torch.randn(w.T, 4, 128, device=DEV).half()
    before = w.w.clone()
    want = w.cache.attend(0, w.batch, q, out=torch.zeros_like(q), add_weights=True)
    weights = w.w.clone()
    w.w.copy_(before)
    got = w.cache.attend(0, w.batch, q, out=torch.zeros_like(q), window=window, add_weights=True)
    assert torch.equal(got, want) and torch.equal(w.w, weights) and (got != 0).any()
    few = World([1, 3, 60], [4, 9, 2], 2, 128, 16, "int8")
    q = torch.randn(few.T, 4, 128, device=DEV).half()
    assert torch.equal(few.cache.attend(0, few.batch, q, out=torch.zeros_like(q)),
                       few.cache.attend(0, few.batch, q, out=torch.zeros_like(q), window=window))


def test_sizes_beyond_32_bits_are_refused():
    # the C interface takes ints: 2^32 + 5 would arrive as 5
    sl = _sl()
    w = World([40], [1], 2, 64, 16, "int8")
    q = torch.randn(w.T, 4, 64, device=DEV).half()
    b = w.batch
    big = 2 ** 32 + 5
    for call in (lambda: w.cache.attend(0, b, q, window=big), lambda: w.cache.attend(0, b, q, window=2 ** 31),
                 lambda: sl.KvBatch(b.page_table, b.kv_len, b.q_start, b.q_len, big),
                 lambda: w.cache.evict(0, b, big, 4), lambda: w.cache.read(0, b, torch.float16, big)):
        with pytest.raises(RuntimeError, match="2.31 or more"):
            call()
    for call in (lambda: w.cache.attend(0, b, q, window=-1), lambda: w.cache.evict(0, b, 16, -1), lambda: w.cache.evict(0, b, 16, 1, sink=-1)):
        with pytest.raises(RuntimeError, match="must not be negative"):
            call()


def test_nan_and_inf_in_q_stay_in_their_rows():
    w = World([100, 500], [1, 2], 2, 128, 16, "int8")
    g = torch.Generator().manual_seed(0)
    clean = torch.randn(w.T, 8, 128, generator=g).half().to(DEV)
    want, _ = _run_attend(w, 8, "fp16", q=clean)
    q = clean.clone()
    q[w.starts[0], 3, 5] = math.nan
    q[w.starts[1] + 1, 0, 0] = math.inf
    out = w.cache.attend(0, w.batch, q)
    own = w.own_rows()
    bad = torch.zeros(w.T, 8, dtype=torch.bool, device=DEV)
    bad[w.starts[0], 3] = bad[w.starts[1] + 1, 0] = True
    assert torch.isnan(out[bad]).all()
    assert torch.equal(out[own[:, None] & ~bad], want[own[:, None] & ~bad])


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_extreme_scales_and_queries(kind):
    w = World([200, 90], [1, 1], 1, 128, 16, kind)
    w.vs[w.table[0, 0]] *= 1e-6       # pages whose values differ by many powers of two
    w.vs[w.table[0, 3]] *= 3e3
    w.vs[w.table[1, 1]] = 0.0
    w.ks[w.table[1, 2]] = 0.0
    g = torch.Generator().manual_seed(3)
    q = torch.randn(w.T, 4, 128, generator=g).bfloat16().to(DEV)
    q[:, 1] *= 2.0 ** -60             # far below f16's range, and far above
    q[:, 2] *= 2.0 ** 18
    q[:, 3] = 0.0
    out = torch.full_like(q, 7.0)
    lse = torch.full((w.T, 4), 7.0, device=DEV)
    w.cache.attend(0, w.batch, q, out=out, lse=lse, scale=2.0 ** -18)
    _check_attend(w, q, out, lse, None, None, 0, 2.0 ** -18)


def _check_rows(w, q, out, window=0, without=()):
    """As _check_attend, row by row: p vs is held to 2^-31 of a reference that is at most 2^9 times the largest v scale of the
    keys that lie together, so a key adds at most 2^-22 |v|; |v| of the keys that the row sees, those of the pages in `without`
    (whose p are next to 0) aside."""
    kv, vv = ref.values(w.k8), ref.values(w.v8)
    u = torch.finfo(q.dtype).eps / 2
    for i, (n, m, r0) in enumerate(zip(w.lens, w.new, w.starts)):
        k = ref.dense(kv, w.ks.double(), w.table[i], n)
        v = ref.dense(vv, w.vs.double(), w.table[i], n)
        o, _, _, mag, size = ref.attend(k, v, q[r0:r0 + m].double(), window, w.d ** -0.5)
        ds = 2.0 ** -22 * (w.d / 16 + 8) * size
        at, last = torch.arange(n, device=DEV), n - m + torch.arange(m, device=DEV)[:, None]
        seen = (at <= last) & ((at > last - window) if window else torch.ones_like(at <= last))
        heard = torch.tensor([int(w.table[i, pos // w.page]) not in without for pos in range(n)], device=DEV)
        most = torch.where(seen & heard, v.abs().amax((0, 2)), 0.0).amax(1)                        # [rows]
        tol = u * o.abs() + (2.0 ** -11 + 4 * ds + 2.0 ** -19) * mag + 2.0 ** -25 + (n * 2.0 ** -22 * most)[:, None, None]
        off = (out[r0:r0 + m].double() - o).abs() / tol
        assert float(off.max()) <= 1, (i, float(off.max()), off.amax((1, 2)).argmax())


@pytest.mark.parametrize("d,page,kind", [(128, 16, "int8"), (64, 64, "e4m3"), (128, 128, "int8")])
@pytest.mark.parametrize("more", [1e5, 2.0 ** 110])
def test_chunks_pay_nothing_for_pages_they_do_not_see(d, page, kind, more):
    # one page of far larger values: rows before it, and rows whose window has passed it, give the same bits without it
    w = World([900, 640, 200], [330, 640, 70], 2, d, page, kind)
    q = torch.randn(w.T, 8, d, device=DEV).bfloat16()
    for window in (0, 100):
        want = w.cache.attend(0, w.batch, q, window=window)
        loud = [int(w.table[0, 640 // page]), int(w.table[1, 256 // page]), int(w.table[2, 128 // page])]
        old = w.vs[loud].clone()
        w.vs[loud] *= more
        got = w.cache.attend(0, w.batch, q, window=window)
        for i, first in enumerate((640, 256, 128)):
            n, m, r0 = w.lens[i], w.new[i], w.starts[i]
            behind = min(first + page, n) + (window if window else n) - 1
            for j in range(m):
                if n - m + j < first or n - m + j >= behind:
                    assert torch.equal(got[r0 + j], want[r0 + j]), (i, j)
        if more < 1e6:
            _check_rows(w, q, got, window)
        assert torch.isfinite(got[w.own_rows()].float()).all()
        w.vs[loud] = old


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("at", [0, 3])
def test_chunks_recover_from_large_values_of_no_weight(d, at):
    # a page of large values (128 keys) that no query attends to: the others keep their bits
    w = World([900], [200], 1, d, 128, "int8")
    q = torch.randn(w.T, 4, d, device=DEV).abs().bfloat16()
    p = int(w.table[0, at])
    w.k8[p] = -127
    w.ks[p] = 100.0 / 127 / d ** 0.5 / 0.7        # scores of -100 or so
    w.vs[p] *= 1e8
    _check_rows(w, q, w.cache.attend(0, w.batch, q), without=(p,))


@pytest.mark.parametrize("hq,hkv,d,page,kind", [(8, 2, 128, 16, "int8"), (4, 1, 64, 16, "e4m3"), (4, 2, 64, 32, "int8"),
                                                (4, 1, 256, 16, "int8"), (2, 2, 128, 16, "e4m3")])
@pytest.mark.parametrize("more", [1e5, 2.0 ** 110])
def test_rows_pay_nothing_for_pages_they_do_not_see(hq, hkv, d, page, kind, more):
    # a few tokens at once: a page of far larger values that the window of the later ones has passed, or that the earlier ones
    # do not reach; the same bits as without it
    w = World([900, 333], [6, 6], hkv, d, page, kind)
    q = torch.randn(w.T, hq, d, device=DEV).bfloat16()
    for window in (0, 98, 107):        # the first token's first key is the third from a page's end
        want = w.cache.attend(0, w.batch, q, window=window)
        for i, n in enumerate(w.lens):
            begins = (n - 6 + 1 - window if window else 0) // page     # the page of the first key that the first token sees
            for b in {max(begins, 0), (n - 1) // page}:
                old = w.vs[int(w.table[i, b])].clone()
                w.vs[int(w.table[i, b])] *= more
                got = w.cache.attend(0, w.batch, q, window=window)
                w.vs[int(w.table[i, b])] = old
                assert torch.isfinite(got[w.own_rows()].float()).all()
                for j in range(6):
                    pos = n - 6 + j
                    sees = pos >= b * page and (not window or pos - window < (b + 1) * page - 1)
                    if not sees:
                        assert torch.equal(got[w.starts[i] + j], want[w.starts[i] + j]), (window, i, b, j)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 5])
@pytest.mark.parametrize("io", ["fp16", "bf16"])
@pytest.mark.parametrize("at", [0, 7, 55])
def test_rows_recover_from_large_values_of_no_weight(d, new, io, at):
    w = World([900], [new], 1, d, 16, "int8")
    q = torch.randn(w.T, 4, d, device=DEV).abs().to(_io(io))
    p = int(w.table[0, at])
    w.k8[p] = -127
    w.ks[p] = 100.0 / 127 / d ** 0.5 / 0.7        # scores of -100 or so
    w.vs[p] *= 1e8
    _check_rows(w, q, w.cache.attend(0, w.batch, q), without=(p,))


@pytest.mark.parametrize("lens,new,hq,hkv,d,page,kind,window", [
    ([18, 505, 1517, 24, 56], [17, 5, 17, 8, 40], 18, 2, 64, 64, "e4m3", 200),
    ([700, 333, 2000], [1, 3, 2], 8, 2, 128, 16, "int8", 100),
    ([700, 90], [4, 7], 4, 1, 256, 16, "int8", 33),
    ([700, 90], [1, 1], 8, 1, 128, 32, "e4m3", 0),
    ([900, 640], [300, 70], 8, 1, 128, 16, "int8", 200),
    ([900, 640], [300, 70], 2, 1, 64, 128, "e4m3", 0),
])
@pytest.mark.parametrize("span", [2, 12, 60])
def test_scales_that_differ_from_page_to_page(lens, new, hq, hkv, d, page, kind, window, span):
    w = World(lens, new, hkv, d, page, kind)
    g = torch.Generator().manual_seed(span)
    w.vs.mul_((2.0 ** torch.randint(-span, span + 1, w.vs.shape, generator=g)).to(DEV))
    q = torch.randn(w.T, hq, d, generator=g).bfloat16().to(DEV)
    _check_rows(w, q, w.cache.attend(0, w.batch, q, window=window), window)


def test_rows_that_are_not_there_cost_no_time():
    # 64 rows of a 256-row tile: those that see no key must not send their warps the long way (it took twice the time of 256)
    def took(new):
        w = World([4096], [new], 1, 128, 128, "int8", track=False)
        q = torch.randn(w.T, 8, 128, device=DEV).bfloat16()
        times = []
        for _ in range(12):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            w.cache.attend(0, w.batch, q)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return sorted(times)[len(times) // 2]

    assert took(8) < 1.5 * took(32)


def test_strided_rows_and_scale():
    sl = _sl()
    w = World([300, 20], [1, 3], 2, 64, 16, "int8")
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(w.T, 3 * 4 * 64 + 8, generator=g).half().to(DEV)
    q = wide[:, 256:512].view(w.T, 4, 64)
    home = torch.full((w.T, 2 * 256), 7.0, dtype=torch.float16, device=DEV)
    out = home[:, 256:].view(w.T, 4, 64)
    w.cache.attend(0, w.batch, q, out=out, scale=0.3)
    _check_attend(w, q, out, None, None, None, 0, 0.3)
    assert (home[:, :256] == 7.0).all()
    with pytest.raises(RuntimeError, match="contiguous heads"):
        w.cache.attend(0, w.batch, q.transpose(1, 2))
    with pytest.raises(RuntimeError, match="aligned"):
        w.cache.attend(0, w.batch, wide[:, 1:257].view(w.T, 4, 64))
    assert isinstance(w.cache, sl.KvCache8)


def test_results_do_not_depend_on_timing():
    w = World([4000, 900, 17, 2500], [1, 3, 2, 1], 2, 128, 32, "int8")
    q = torch.randn(w.T, 16, 128, device=DEV, dtype=torch.bfloat16)
    w.w.zero_()
    first = (w.cache.attend(0, w.batch, q, out=torch.zeros_like(q), add_weights=True), w.w.clone())
    for _ in range(5):
        w.w.zero_()
        out = w.cache.attend(0, w.batch, q, out=torch.zeros_like(q), add_weights=True)
        assert torch.equal(out, first[0]) and torch.equal(w.w, first[1])


@pytest.mark.parametrize("lens,new,hq,hkv,d", [
    ([3000, 2500, 700, 90] * 4, [6, 5, 7, 1] * 4, 16, 2, 128),     # up to 56 rows: four blocks of 16
    ([3000, 2500, 700, 90] * 2, [6, 5, 7, 1] * 2, 8, 1, 256),      # seven blocks of eight
    ([900, 300], [200, 70], 8, 1, 128),                            # scores computed again
])
def test_weights_do_not_depend_on_timing(lens, new, hq, hkv, d):
    # added to what was there: with three addends or more their order would show
    w = World(lens, new, hkv, d, 32, "int8")
    q = torch.randn(w.T, hq, d, device=DEV, dtype=torch.bfloat16)
    before, first = w.w.clone(), None
    for _ in range(25):
        w.w.copy_(before)
        w.cache.attend(0, w.batch, q, add_weights=True)
        first = w.w.clone() if first is None else first
        assert torch.equal(w.w, first)
    _run_attend(w, hq, "fp16", weights=True)


def test_bad_tables_are_skipped_and_reported():
    sl = _sl()
    # the kernels check every entry before they use it: a bad sequence's rows stay as they are, a bad page's keys drop out
    w = World([100, 80, 60], [1, 1, 1], 2, 128, 16, "int8")
    q = torch.randn(w.T, 4, 128, device=DEV).half()

    def run(table=None, kv=None, start=None, ql=None, max_q=1):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        b = sl.KvBatch((w.table if table is None else table).to(DEV), i32(kv or w.lens), i32(start or w.starts), i32(ql or w.new), max_q)
        out = w.cache.attend(0, b, q, out=torch.full_like(q, 7.0), add_weights=True)
        kept = w.cache.evict(0, b, 256, 4)
        k, v = w.cache.read(0, b, torch.float16, 8)
        torch.cuda.synchronize()
        assert b.status() & 2
        with pytest.raises(RuntimeError, match="bad table entry"):
            b.check()
        return out, kept, k

    good = w.cache.attend(0, w.batch, q, out=torch.full_like(q, 7.0))
    for kw in (dict(kv=[113, 80, 60]), dict(kv=[-1, 80, 60]), ):
        out, kept, k = run(**kw)
        assert (out[w.starts[0]] == 7.0).all() and torch.equal(out[w.starts[1]], good[w.starts[1]])
        assert (kept[0] == -1).all() and (k[0] == 0).all()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    for kw in (dict(start=[w.T, w.starts[1], w.starts[2]]), dict(start=[-1, w.starts[1], w.starts[2]]), dict(ql=[2, 1, 1]),
               dict(ql=[-1, 1, 1])):
        b = sl.KvBatch(w.table.to(DEV), i32(w.lens), i32(kw.get("start", w.starts)), i32(kw.get("ql", w.new)), 1)
        before = w.k8.view(torch.uint8).clone()
        out = w.cache.attend(0, b, q, out=torch.full_like(q, 7.0))
        assert torch.equal(out[w.starts[1:]], good[w.starts[1:]]) and b.status() == 2
        own = torch.zeros(w.T, dtype=torch.bool)
        own[w.starts[1:]] = True
        assert (out[~own.to(DEV)] == 7.0).all()
        x = torch.randn(w.T, 2, 128, device=DEV).half()
        w.cache.append(0, b, x, x)
        torch.cuda.synchronize()
        changed = (w.k8.view(torch.uint8) != before).flatten(1).any(1).nonzero().flatten().tolist()
        assert set(changed) <= {int(w.table[1, 4]), int(w.table[2, 3])}
        w.k8.view(torch.uint8).copy_(before)
        w = World([100, 80, 60], [1, 1, 1], 2, 128, 16, "int8")
    bad = w.table.clone()
    bad[0, 2] = w.cache.n_pages
    bad[1, 0] = -1
    out, kept, _ = run(table=bad)
    assert torch.isfinite(out.float()).all() and torch.equal(out[w.starts[2]], good[w.starts[2]])
    assert not torch.equal(out[w.starts[0]], good[w.starts[0]])


@pytest.mark.parametrize("bound", [80, 77, 81, 0, 10 ** 9])
def test_bound_of_the_lengths(bound):
    # 80 tokens are five pages of 16: a bound of 77 reaches as far, one of 81 takes a sixth page in, 0 leaves no key
    sl = _sl()
    w = World([100, 80, 60], [1, 1, 1], 2, 128, 16, "int8")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    q = torch.randn(w.T, 4, 128, device=DEV).half()
    good = w.cache.attend(0, w.batch, q, out=torch.full_like(q, 7.0))
    b = sl.KvBatch(w.batch.page_table, i32(w.lens), i32(w.starts), i32(w.new), 1, bound)
    out = w.cache.attend(0, b, q, out=torch.full_like(q, 7.0), add_weights=True)
    for i, n in enumerate(w.lens):
        inside = n <= -(-bound // 16) * 16
        assert torch.equal(out[w.starts[i]], good[w.starts[i]] if inside else torch.full_like(q[0], 7.0)), i
    assert b.status() == (0 if bound >= 100 else 2)
    kept = w.cache.evict(0, b, 50, 4)
    for i, n in enumerate(w.lens):
        assert bool((kept[i] >= 0).all()) == (n <= -(-bound // 16) * 16), i


def test_empty_batches():
    sl = _sl()
    w = World([30], [1], 2, 64, 16, "int8")
    none = sl.KvBatch(torch.zeros((0, 4), dtype=torch.int64, device=DEV), *[torch.zeros(0, dtype=torch.int32, device=DEV)] * 3, 0)
    q = torch.randn(0, 4, 64, device=DEV).half()
    assert w.cache.attend(0, none, q).shape == q.shape
    w.cache.append(0, none, q[:, :2], q[:, :2])
    assert w.cache.evict(0, none, 8, 2).shape == (0, 2, 8)
    assert w.cache.read(0, none, torch.float16, 5)[0].shape == (0, 5, 2, 64)
    idle = World([30, 20], [0, 0], 2, 64, 16, "int8")
    q = torch.randn(idle.T, 4, 64, device=DEV).half()
    out = torch.full_like(q, 7.0)
    assert (idle.cache.attend(0, idle.batch, q, out=out) == 7.0).all()


def test_sequences_that_share_a_prefix():
    """Two sequences whose first pages are the same: both read them, and their weights gather both sequences' attention."""
    w = World([70, 90, 40], [1, 1, 1], 2, 64, 16, "int8")
    w.table[1, :3] = w.table[0, :3]
    w.batch.page_table.copy_(w.table)
    q = torch.randn(w.T, 4, 64, device=DEV).half()
    before = w.w.clone()
    out = w.cache.attend(0, w.batch, q, out=torch.zeros_like(q), add_weights=True)
    _check_attend(w, q, out, None, None, None)
    want = before.double()
    for i, (n, r) in enumerate(zip(w.lens, w.starts)):
        k = ref.dense(ref.values(w.k8), w.ks.double(), w.table[i], n)
        v = ref.dense(ref.values(w.v8), w.vs.double(), w.table[i], n)
        p = ref.attend(k, v, q[r:r + 1].double(), 0, 64 ** -0.5)[2]
        for pos in range(n):
            want[int(w.table[i, pos // 16]), :, pos % 16] += p[:, pos]
    assert ((w.w.double() - want).abs() <= 2.0 ** -16 * (want + 1)).all()


@pytest.mark.parametrize("new", [1, 130])
def test_negative_and_zero_scale(new):
    w = World([200, 131], [new, new], 2, 128, 32, "e4m3")
    for scale in (-0.2, 0.0):
        q = torch.randn(w.T, 4, 128, device=DEV).half()
        out = w.cache.attend(0, w.batch, q, scale=scale)
        own = w.own_rows()
        full = torch.zeros_like(q)
        full[own] = out[own]
        for i, (n, m, r0) in enumerate(zip(w.lens, w.new, w.starts)):
            k = ref.dense(ref.values(w.k8), w.ks.double(), w.table[i], n)
            v = ref.dense(ref.values(w.v8), w.vs.double(), w.table[i], n)
            o, _, _, mag, _ = ref.attend(k, v, q[r0:r0 + m].double(), 0, scale)
            # as in _check_attend, with the size of the scores from |scale|
            size = float((q[r0:r0 + m].double().abs().sum(-1).max() * k.abs().max()) * abs(scale))
            ds = 2.0 ** -22 * 16 * size
            tol = 2.0 ** -11 * o.abs() + (2.0 ** -11 + 4 * ds + 2.0 ** -19) * mag + 2.0 ** -25 + n * 2.0 ** -29 * float(v.abs().max())
            assert bool(((full[r0:r0 + m].double() - o).abs() <= tol).all())


def test_pages_beyond_four_gigabytes():
    # 2^32 bytes lie between the first and the last page
    sl = _sl()
    n, hkv, d, page = 66000, 8, 128, 64
    k8 = torch.zeros((n, hkv, page, d), dtype=torch.int8, device=DEV)
    v8 = torch.zeros_like(k8)
    ks, vs = torch.zeros((n, hkv), device=DEV), torch.zeros((n, hkv), device=DEV)
    wt = torch.zeros((n, hkv, page), device=DEV)
    cache = sl.KvCache8.from_buffers([k8], [v8], [ks], [vs], [wt])
    table = torch.tensor([[65999, 3], [0, 65998]], dtype=torch.int64)
    lens, new = [100, 100], [100, 100]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    batch = sl.KvBatch(table.to(DEV), i32(lens), i32([0, 100]), i32(new), 100)
    x, y = (torch.randn(200, hkv, d, device=DEV).half() for _ in range(2))
    cache.append(0, batch, x, y)
    for t, x8, s in ((x, k8, ks), (y, v8, vs)):
        zero = torch.zeros((4, hkv, page, d), dtype=torch.int8, device=DEV)
        small = {65999: 0, 3: 1, 0: 2, 65998: 3}
        tab = torch.tensor([[small[int(p)] for p in r] for r in table])
        val, sc = ref.append(zero, torch.zeros(4, hkv, device=DEV), tab, lens, [0, 100], new, t.double(), "int8")
        for p, i in small.items():
            assert torch.equal(x8[p].double(), val[i]) and torch.equal(s[p].double(), sc[i])
    w = World.__new__(World)
    w.lens, w.new, w.starts, w.page, w.hkv, w.d, w.table = lens, [1, 1], [0, 1], page, hkv, d, torch.tensor([[0, 1], [2, 3]])
    w.T = 2
    pick = [65999, 3, 0, 65998]
    w.k8, w.v8, w.ks, w.vs = k8[pick], v8[pick], ks[pick], vs[pick]
    q = torch.randn(2, 16, d, device=DEV).half()
    dec = sl.KvBatch(table.to(DEV), i32(lens), i32([0, 1]), i32([1, 1]), 1)
    out = cache.attend(0, dec, q, add_weights=True)
    _check_attend(w, q, out, None, wt[pick], torch.zeros(4, hkv, page, device=DEV))
    kept = cache.evict(0, dec, 64, 10)
    assert (kept[:, :, -10:] == torch.arange(90, 100, device=DEV)).all()


# ---- append and read ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("lens,new,hkv,d,page,kind,io", [
    ([1, 16, 17, 40], [1, 1, 1, 1], 2, 128, 16, "int8", "fp16"),
    ([1, 16, 17, 40], [1, 1, 1, 1], 2, 128, 16, "e4m3", "bf16"),
    ([5, 100, 64, 333, 20], [5, 2, 64, 300, 0], 3, 64, 32, "int8", "bf16"),
    ([130, 128, 250], [130, 1, 7], 1, 256, 128, "e4m3", "fp16"),
    ([130, 128, 250], [130, 1, 7], 2, 256, 64, "int8", "fp16"),
    ([60 + i for i in range(40)], [1 + i % 3 for i in range(40)], 4, 128, 64, "int8", "fp16"),
])
def test_append_without_rotary_is_exact(lens, new, hkv, d, page, kind, io):
    w = World(lens, new, hkv, d, page, kind)
    g = torch.Generator().manual_seed(4)
    x, y = (torch.randn(w.T, hkv, d, generator=g).to(_io(io)).to(DEV) for _ in range(2))
    x[:, :, ::7] *= 6                                   # some scales grow, some do not
    x[w.starts[0]] = 0
    k0, v0, w0 = w.k8.clone(), w.v8.clone(), w.w.clone()
    want = [ref.append(a, s, w.table, w.lens, w.starts, w.new, t.double(), kind)
            for a, s, t in ((w.k8, w.ks, x), (w.v8, w.vs, y))]
    w.cache.append(0, w.batch, x, y)
    torch.cuda.synchronize()
    assert w.batch.status() == 0
    for (val, sc), a, was, s in zip(want, (w.k8, w.v8), (k0, v0), (w.ks, w.vs)):
        assert torch.equal(torch.nan_to_num(sc, -1.0), torch.nan_to_num(s.double(), -1.0))
        live = torch.zeros(a.shape[:3], dtype=torch.bool, device=DEV)
        for i, n in enumerate(lens):
            for b in range(-(-n // page)):
                live[int(w.table[i, b]), :, :min(page, n - b * page)] = True
        assert torch.equal(ref.values(a)[live], val[live])
        assert torch.equal(a.view(torch.uint8)[~live], was.view(torch.uint8)[~live])     # everything else as it was
    fresh = torch.zeros_like(w.w, dtype=torch.bool)
    for i, (n, m) in enumerate(zip(lens, new)):
        for pos in range(n - m, n):
            fresh[int(w.table[i, pos // page]), :, pos % page] = True
    assert (w.w[fresh] == 0).all() and torch.equal(w.w[~fresh], w0[~fresh])
    # and back
    first = torch.tensor([max(0, n - 20) for n in lens], dtype=torch.int32, device=DEV)
    for dt in (torch.float16, torch.bfloat16):
        k, v = w.cache.read(0, w.batch, dt, 33, first=first)
        for got, a, s in ((k, w.k8, w.ks), (v, w.v8, w.vs)):
            for i, n in enumerate(lens):
                f = int(first[i])
                m = min(33, n - f)
                full = ref.dense(ref.values(a).float(), s, w.table[i], n)[:, f:f + m].transpose(0, 1)
                assert torch.equal(got[i, :m], full.to(dt)) and (got[i, m:] == 0).all()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_appending_one_by_one(kind):
    """The cache after many small appends: every value within half a step per scale change of what was appended."""
    sl = _sl()
    cache = sl.KvCache8(4, 16, 2, 64, kind=kind, track_weights=True)
    g = torch.Generator().manual_seed(8)
    x = torch.randn(40, 2, 64, generator=g).half().to(DEV) * torch.linspace(0.5, 3, 40, device=DEV)[:, None, None].half()
    table = torch.tensor([[2, 0, 3]], dtype=torch.int64, device=DEV)
    i32 = lambda v: torch.tensor([v], dtype=torch.int32, device=DEV)  # noqa: E731
    val, sc = cache.k[0].clone(), cache.k_scale[0].clone()
    at = 0
    for step in (1, 1, 3, 10, 1, 1, 7, 16):
        b = sl.KvBatch(table, i32(at + step), i32(0), i32(step), step)
        cache.append(0, b, x[at:at + step], x[at:at + step])
        v64, s64 = ref.append(val, sc, table.cpu(), [at + step], [0], [step], x[at:at + step].double(), kind)
        val, sc = v64.float().to(ref.DTYPE[kind]), s64.float()
        at += step
        b.check()
    assert torch.equal(cache.k[0].view(torch.uint8), val.view(torch.uint8)) and torch.equal(cache.k_scale[0], sc)
    assert torch.equal(cache.v[0].view(torch.uint8), val.view(torch.uint8))
    got, _ = cache.read(0, b, torch.float16, 40)
    top = x.abs().max()
    assert (got[0] - x).abs().max() <= top * (0.5 / 127 * 6 if kind == "int8" else 2.0 ** -4 * 6)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("new", [2, 9])          # a warp's page, and the whole CTA's
@pytest.mark.parametrize("top", [0.0, 1.0])      # new values: all 0, and not
def test_a_scale_below_the_normal_numbers_counts_as_zero(kind, new, top):
    lens = [new + 5, 20 + new]
    w = World(lens, [new, new], 2, 64, 16, kind)
    firsts = [(int(w.table[i, (n - new) // 16]), (n - new) % 16) for i, n in enumerate(lens)]    # pages with older tokens
    for p, _ in firsts:
        w.ks[p], w.vs[p] = 2.0 ** -127, 2.0 ** -149
    x = torch.randn(w.T, 2, 64, device=DEV).half() * top
    w.cache.append(0, w.batch, x, x)
    torch.cuda.synchronize()
    assert w.batch.status() == 0
    for (p, n0), n, r0 in zip(firsts, lens, w.starts):
        m = min(16, n0 + new) - n0                # new tokens of that page
        y = x[r0:r0 + m].transpose(0, 1).double()
        s = ref.scale_of(y.abs().amax((1, 2)), kind)
        for x8, sc in ((w.k8, w.ks), (w.v8, w.vs)):
            assert torch.equal(sc[p].double(), s)
            assert (ref.values(x8)[p, :, :n0] == 0).all()
            assert torch.equal(ref.values(x8)[p, :, n0:n0 + m], ref.nearest(y / torch.where(s > 0, s, 1.0)[:, None, None], kind))
    k, v = w.cache.read(0, w.batch, torch.float16, max(lens))
    out = w.cache.attend(0, w.batch, torch.randn(w.T, 4, 64, device=DEV).half())
    assert torch.isfinite(k).all() and torch.isfinite(v).all() and torch.isfinite(out[w.own_rows()]).all()


def test_nonfinite_values_are_stored_finite_and_reported():
    w = World([20, 33], [4, 33], 2, 64, 16, "int8")
    x = torch.randn(w.T, 2, 64, device=DEV).half()
    y = x.clone()
    clean = x.clone()
    r = w.starts[1]
    x[r, 0, 3], x[r + 20, 1, 0], x[r + 20, 1, 1] = math.nan, math.inf, -math.inf
    clean[r, 0, 3] = clean[r + 20, 1, 0] = clean[r + 20, 1, 1] = 0
    want, sc = ref.append(w.k8, w.ks, w.table, w.lens, w.starts, w.new, clean.double(), "int8")
    w.cache.append(0, w.batch, x, y)
    assert w.batch.status() == 16
    p = [int(t) for t in w.table[1]]
    assert w.k8[p[0], 0, 0, 3] == 0 and w.k8[p[1], 1, 4, 0] == 127 and w.k8[p[1], 1, 4, 1] == -127
    want[p[1], 1, 4, 0], want[p[1], 1, 4, 1] = 127, -127
    assert torch.equal(w.k8[p].double()[:2], want[p][:2]) and torch.equal(w.ks[p].double(), sc[p])


@pytest.mark.parametrize("layout,rot,d,io", [("half", 128, 128, "fp16"), ("half", 32, 128, "bf16"), ("interleaved", 64, 64, "fp16"),
                                             ("interleaved", 96, 128, "bf16"), ("half", 96, 256, "fp16")])
def test_append_with_rotary(layout, rot, d, io):
    sl = _sl()
    w = World([40, 70, 16, 500], [1, 70, 3, 20], 2, d, 16, "int8")
    table = sl.RotaryTable(d, rot, layout=layout)
    pos = torch.arange(w.T, device=DEV) * 97 + 11
    q, x, y = (torch.randn(w.T, h, d, device=DEV).to(_io(io)) for h in (6, 2, 2))
    q0, x0 = q.clone(), x.clone()
    turned = ref.rotate(x.double(), pos, table.inv_freq, 1.0, layout)
    want, sc = ref.append(w.k8, w.ks, w.table, w.lens, w.starts, w.new, turned, "int8")
    q_out = torch.full_like(q, 7.0)
    got = w.cache.append(0, w.batch, x, y, q=q, rope=(table, pos), q_out=q_out)
    assert got is q_out and torch.equal(q, q0) and torch.equal(x, x0)
    own = w.own_rows()
    tq = ref.rotate(q.double(), pos, table.inv_freq, 1.0, layout)
    u = torch.finfo(q.dtype).eps / 2
    size = q.double().abs().amax(-1, keepdim=True) * 2
    assert ((q_out.double() - tq).abs() <= u * tq.abs() + 2.0 ** -20 * size)[own].all() and (q_out[~own] == 7.0).all()
    # scales: the maximum of values within 2^-20 of theirs; values: within half a step and that
    for i, n in enumerate(w.lens):
        for b in range((n - w.new[i]) // 16, -(-n // 16)):
            p, m = int(w.table[i, b]), min(16, n - b * 16)
            s = w.ks[p].double()
            assert ((s - sc[p]).abs() <= 2.0 ** -19 * 8 / 127).all()
            assert ((w.k8[p, :, :m].double() - want[p, :, :m]).abs() <= 1).all()
            n0 = max(0, n - w.new[i] - b * 16)
            r0 = w.starts[i] + max(0, b * 16 - (n - w.new[i]))
            x64 = turned[r0:r0 + m - n0].transpose(0, 1)
            off = (w.k8[p, :, n0:m].double() * s[:, None, None] - x64).abs()
            assert (off <= s[:, None, None] * 0.5 + 2.0 ** -18 * 8).all()
    again = w.cache.append(0, w.batch, x, y, q=q, rope=(table, pos))        # in place
    assert again is q and torch.equal(q[own], q_out[own])


# ---- rotary -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("T", [1, 7, 33, 1000])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,rot,scaling", [(128, 128, None), (128, 64, {"type": "yarn", "factor": 16.0, "original_max_position": 4096}),
                                           (64, 16, {"type": "ntk", "factor": 3.0}), (256, 240, None)])
def test_rotary(T, layout, d, rot, scaling):
    sl = _sl()
    table = sl.RotaryTable(d, rot, layout=layout, scaling=scaling)
    g = torch.Generator().manual_seed(T)
    pos = torch.randint(0, 1 << 20, (T,), generator=g).to(DEV)
    pos[0] = 0
    for io in (torch.float16, torch.bfloat16):
        q, k = torch.randn(T, 5, d, generator=g).to(io).to(DEV), torch.randn(T, 2, d + 8, generator=g).to(io).to(DEV)[:, :, :d].contiguous()
        wide = torch.full((T, 2 * d + 16), 7.0, dtype=io, device=DEV)
        k_out = wide[:, 16:].view(T, 2, d)
        qo, ko = sl.rotary(table, pos, q, k, q_out=torch.empty_like(q), k_out=k_out)
        u = torch.finfo(io).eps / 2
        for x, y in ((q, qo), (k, ko)):
            want = ref.rotate(x.double(), pos, table.inv_freq, table.factor, layout)
            tol = u * want.abs() + 2.0 ** -20 * 2 * table.factor * x.double().abs().amax(-1, keepdim=True)
            assert ((y.double() - want).abs() <= tol).all()
            assert torch.equal(y[..., rot:], x[..., rot:])
        assert (wide[:, :16] == 7.0).all()
        back, none = sl.rotary(table, pos, qo.clone(), inverse=True)
        assert none is None
        want = ref.rotate(qo.double(), pos, table.inv_freq, table.factor, layout, inverse=True)
        assert ((back.double() - want).abs() <= u * want.abs() + 2.0 ** -18 * 2 * x.double().abs().amax()).all()
        same, _ = sl.rotary(table, pos, q.clone())
        assert torch.equal(same, qo)


def test_rotary_matches_the_cosine_rows_of_the_lora_path():
    """The half layout over whole heads is what ``lora_get_qkv(rope=(cos, sin))`` computes from rounded rows: the two
    agree to the rounding of those rows."""
    sl = _sl()
    table = sl.RotaryTable(128)
    pos = torch.arange(50, device=DEV) * 13
    q = torch.randn(50, 4, 128, device=DEV).half()
    y, _ = sl.rotary(table, pos, q, q_out=torch.empty_like(q))
    a = pos.double()[:, None] * torch.tensor(table.inv_freq, dtype=torch.float64, device=DEV)
    c, s = a.cos().half().double()[:, None], a.sin().half().double()[:, None]
    lo, hi = q[..., :64].double(), q[..., 64:].double()
    want = torch.cat([lo * c - hi * s, lo * s + hi * c], -1)
    size = torch.cat([lo.abs() + hi.abs()] * 2, -1)
    assert ((y.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -11 * size + 2.0 ** -18 * size).all()


def test_rotary_refusals_on_the_device():
    sl = _sl()
    table = sl.RotaryTable(64)
    q = torch.randn(4, 2, 64, device=DEV).half()
    pos = torch.arange(4, device=DEV)
    for bad in (dict(positions=pos.int()), dict(positions=pos[:3]), dict(q=q.float()), dict(q=q[:, :, :32]),
                dict(k=q[:3]), dict(q_out=q[:, :1]), dict(k_out=q)):
        kw = dict(table=table, positions=pos, q=q)
        kw.update(bad)
        with pytest.raises(RuntimeError):
            sl.rotary(**kw)


# ---- eviction -----------------------------------------------------------------------------------------------------

def _check_evict(w, before, kept, budget, recent, sink, dest_rows):
    k0, v0, ks0, vs0, w0 = before
    touched = torch.zeros(w.k8.shape[:3], dtype=torch.bool, device=DEV)
    scaled = torch.zeros(w.ks.shape, dtype=torch.bool, device=DEV)
    for i, n in enumerate(w.lens):
        pages = w.table[i][: -(-n // w.page)].to(DEV)
        wt = w0[pages].transpose(0, 1).reshape(w.hkv, -1)[:, :n]
        for h in range(w.hkv):
            keep = ref.kept(wt[h].tolist(), n, budget, recent, sink)
            assert kept[i, h].tolist() == keep + [-1] * (budget - len(keep)), (i, h)
            for x0, s0, x8, s in ((k0, ks0, w.k8, w.ks), (v0, vs0, w.v8, w.vs)):
                for p, (q, sc) in ref.move(ref.values(x0), s0, w.table[i].tolist(), keep, h, dest_rows[i], w.kind).items():
                    assert torch.equal(ref.values(x8[p, h, : q.size(0)]), q), (i, h, p)
                    assert float(s[p, h]) == float(sc)
                    touched[p, h, : q.size(0)] = True
                    scaled[p, h] = True
            for j, src in enumerate(keep):
                a, b = float(w.w[int(dest_rows[i][j // w.page]), h, j % w.page]), float(wt[h, src])
                assert a == b or (a != a and b != b)
    for x0, x8 in ((k0, w.k8), (v0, w.v8)):
        assert torch.equal(x0.view(torch.uint8)[~touched], x8.view(torch.uint8)[~touched])
    assert torch.equal(torch.nan_to_num(ks0, -1.0)[~scaled], torch.nan_to_num(w.ks, -1.0)[~scaled])
    assert torch.equal(torch.nan_to_num(w0[~touched], -5.0), torch.nan_to_num(w.w[~touched], -5.0))


@pytest.mark.parametrize("lens,hkv,d,page,kind,budget,recent,sink", [
    ([100, 33, 16, 0, 200], 2, 64, 16, "int8", 48, 10, 2),
    ([100, 33, 16, 0, 200], 2, 128, 16, "e4m3", 37, 37, 0),
    ([300, 129], 1, 128, 64, "int8", 100, 0, 0),
    ([300, 500], 3, 256, 32, "int8", 129, 1, 128),
    ([700, 260], 1, 128, 128, "e4m3", 200, 50, 4),
    ([150, 90], 2, 256, 128, "int8", 64, 5, 0),
    ([3000], 1, 64, 32, "int8", 1, 0, 0),
    ([40], 1, 64, 16, "int8", 1, 1, 0),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict(lens, hkv, d, page, kind, budget, recent, sink, in_place):
    sl = _sl()
    per = -(-budget // page)
    w = World(lens, [0] * len(lens), hkv, d, page, kind, spare=per * len(lens))
    g = torch.Generator().manual_seed(9)
    w.w.copy_(torch.randint(0, 40, w.w.shape, generator=g).float().to(DEV) / 8)      # many ties
    w.w[int(w.table[0, 0]), 0, 3] = math.nan
    w.w[int(w.table[0, 0]), 0, 5] = math.inf
    w.w[int(w.table[0, 0]), 0, 6] = -1.0
    w.w[int(w.table[0, 0]), 0, 7] = -0.0
    before = [t.clone() for t in (w.k8, w.v8, w.ks, w.vs, w.w)]
    rows = [w.free[i * per:(i + 1) * per] for i in range(len(lens))]
    dest = None
    if not in_place:
        i32 = torch.zeros(len(lens), dtype=torch.int32, device=DEV)
        dest = sl.KvBatch(torch.tensor(rows, dtype=torch.int64, device=DEV), i32, i32, i32, 0)
    kept = w.cache.evict(0, w.batch, budget, recent, sink=sink, dest=dest)
    torch.cuda.synchronize()
    assert w.batch.status() == 0
    _check_evict(w, before, kept, budget, recent, sink, [w.table[i].tolist() for i in range(len(lens))] if in_place else rows)


def test_evict_long_sequence():
    """More candidates than fit the shared memory of the selection, all kinds of weights."""
    sl = _sl()
    n, budget = 50000, 700
    w = World([n], [0], 1, 64, 128, "int8", spare=6)
    g = torch.Generator().manual_seed(10)
    w.w.copy_((torch.rand(w.w.shape, generator=g) * 2.0 ** torch.randint(-60, 60, w.w.shape, generator=g)).to(DEV))
    before = [t.clone() for t in (w.k8, w.v8, w.ks, w.vs, w.w)]
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    dest = sl.KvBatch(torch.tensor([w.free], dtype=torch.int64, device=DEV), zero, zero, zero, 0)
    kept = w.cache.evict(0, w.batch, budget, 100, sink=3, dest=dest)
    _check_evict(w, before, kept, budget, 100, 3, [w.free])


# ---- used together ------------------------------------------------------------------------------------------------

def test_streams_and_graphs():
    sl = _sl()
    w = World([300, 45, 800], [1, 1, 1], 2, 128, 16, "int8")
    table = sl.RotaryTable(128)
    pos = torch.tensor(w.lens, device=DEV).repeat(w.T)[: w.T].contiguous() - 1
    q, x, y = (torch.randn(w.T, h, 128, device=DEV).half() for h in (8, 2, 2))
    out, q_out = torch.zeros_like(q), torch.zeros_like(q)

    def step():
        w.cache.append(0, w.batch, x, y, q=q, rope=(table, pos), q_out=q_out)
        w.cache.attend(0, w.batch, q_out, out=out, add_weights=True)

    start = [t.clone() for t in (w.k8, w.v8, w.ks, w.vs, w.w)]

    def reset():
        for t, s in zip((w.k8, w.v8, w.ks, w.vs, w.w), start):
            t.view(torch.uint8).copy_(s.view(torch.uint8))
        out.zero_()

    step()
    torch.cuda.synchronize()
    want = [t.clone() for t in (out, w.k8.view(torch.uint8), w.ks, w.w)]

    side = torch.cuda.Stream()
    reset()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    assert all(torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float())) for a, b in
               zip((out, w.k8.view(torch.uint8), w.ks, w.w), want))

    reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        reset()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float())) for a, b in
                   zip((out, w.k8.view(torch.uint8), w.ks, w.w), want))
    # the tables are read on the device: another step's lengths need no new capture
    w.batch.kv_len.copy_(torch.tensor([299, 44, 700], dtype=torch.int32))
    reset()
    graph.replay()
    torch.cuda.synchronize()
    w.lens = [299, 44, 700]
    _check_attend(w, q_out, out, None, None, None)


def test_calls_run_on_the_device_of_their_tensors(monkeypatch):
    # as on a machine with several GPUs: whatever goes by the current device happens with the tensors' one made current
    from slora_b200 import _lib
    sl = _sl()
    w = World([300, 45], [1, 1], 2, 128, 16, "int8")
    table, pos = sl.RotaryTable(128), torch.zeros(w.T, dtype=torch.int64, device=DEV)
    q, x = torch.randn(w.T, 8, 128, device=DEV).half(), torch.randn(w.T, 2, 128, device=DEV).half()
    inside, called = [0], []

    class Current:
        def __enter__(self):
            inside[0] += 1

        def __exit__(self, *args):
            inside[0] -= 1

    class Library:
        def __getattr__(self, name):
            called.append(name)
            fn = getattr(library, name)

            def call(*args):
                assert inside[0] == 1, name
                return fn(*args)
            return call

    library = _lib.lib
    monkeypatch.setattr(_lib, "lib", Library())
    monkeypatch.setattr(_lib, "device_of", lambda *tensors: Current())
    w.cache.append(0, w.batch, x, x, q=q, rope=(table, pos))
    w.cache.attend(0, w.batch, q, add_weights=True)
    w.cache.read(0, w.batch, torch.float16, 4)
    w.cache.evict(0, w.batch, 32, 4)
    sl.rotary(table, pos, q)
    assert set(called) == {"slora_kv8_append", "slora_kv8_attend_workspace_bytes", "slora_kv8_attend", "slora_kv8_read", "slora_kv8_evict",
                           "slora_rotary"}


def test_two_calls_at_once():
    w = World([2000, 45, 800], [1, 1, 1], 2, 128, 16, "int8")
    qs = [torch.randn(w.T, 8, 128, device=DEV).half() for _ in range(4)]
    want = [w.cache.attend(0, w.batch, q, out=torch.zeros_like(q)) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for q, s in zip(qs, streams):
            with torch.cuda.stream(s):
                got.append(w.cache.attend(0, w.batch, q, out=torch.zeros_like(q)))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_decoding_with_eviction():
    """Prompt, then decode steps with accumulated weights, then eviction and more steps: every step against the cache's
    own content in 64 bits, positions kept by the caller."""
    sl = _sl()
    random.seed(0)
    hq, hkv, d, page = 4, 2, 64, 16
    cache = sl.KvCache8(24, page, hkv, d, kind="int8", track_weights=True)
    table = sl.RotaryTable(d)
    prompt = [50, 23]
    rows = [cache.pages.alloc(6) for _ in prompt]
    pages = torch.stack(rows)
    lens, seen = [0, 0], [0, 0]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731

    def step(new):
        nonlocal lens, seen
        lens = [a + b for a, b in zip(lens, new)]
        start = [0, new[0]]
        pos = torch.cat([torch.arange(s, s + n) for s, n in zip(seen, new)]).to(DEV)
        seen = [a + b for a, b in zip(seen, new)]
        T = sum(new)
        q, k, v = (torch.randn(T, h, d, device=DEV).half() for h in (hq, hkv, hkv))
        batch = sl.KvBatch(pages, i32(lens), i32(start), i32(new), max(new))
        q = cache.append(0, batch, k, v, q=q, rope=(table, pos))
        before = cache.weights[0].clone()
        lse = torch.empty(T, hq, device=DEV)
        out = cache.attend(0, batch, q, lse=lse, add_weights=True)
        w = World.__new__(World)
        w.lens, w.new, w.starts, w.page, w.hkv, w.d, w.table = lens, new, start, page, hkv, d, pages.cpu()
        w.k8, w.v8, w.ks, w.vs = cache.k[0], cache.v[0], cache.k_scale[0], cache.v_scale[0]
        _check_attend(w, q, out, lse, cache.weights[0], before)
        batch.check()
        return batch

    step(prompt)
    for _ in range(10):
        batch = step([1, 1])
    total = cache.weights[0][pages[0][:4]].sum()
    assert abs(float(total) - hq * 60) < 1e-3 * hq * 60           # every query spreads a weight of 1 per head
    kept = cache.evict(0, batch, 32, 8, sink=2)
    assert (kept[0, :, :2].cpu() == torch.tensor([0, 1])).all() and (kept[0, :, -8:].cpu() == torch.arange(52, 60)).all()
    lens = [min(n, 32) for n in lens]
    cache.pages.free(pages[0, 4:].clone())
    for _ in range(3):
        step([1, 1])
    step([5, 2])


@pytest.mark.parametrize("kv,head_dim", [(1024, 128), (256, 64)])
def test_lora_layer_with_the_cache(kv, head_dim):
    """One layer of a decode step through ``LoraBatchOps``: LoRA deltas on the base projections, rotary and append in
    ``lora_get_qkv``, attention, ``lora_get_o``; against the same operators called one by one, and attention in 64 bits."""
    from slora_b200.workloads import build_workload
    sl = _sl()
    wl = build_workload(5, pool_rows=8192, n_adapters=12, decode_tokens=50, hidden=1024, h_kv=kv).to(DEV)
    T, hidden = wl.T, 1024
    ops = sl.LoraBatchOps(wl.a_start, wl.a_len, wl.a_loc, wl.a_scaling, wl.pools_a, wl.pools_b, wl.max_rank)
    ops.prepare(wl.ids)
    g = torch.Generator().manual_seed(2)
    base = [torch.randn(T, n, generator=g).to(wl.dtype).to(DEV) for n in (hidden, kv, kv)]
    table = sl.RotaryTable(head_dim, head_dim // 2, layout="interleaved")
    old = [int(x) for x in torch.randint(0, 90, (T,), generator=g)]
    w = World([n + 1 for n in old], [1] * T, kv // head_dim, head_dim, 16, "int8")
    w.batch.q_start.copy_(torch.arange(T, dtype=torch.int32))
    w.starts, w.T = list(range(T)), T
    pos = torch.tensor(old, dtype=torch.int64, device=DEV)
    start = [t.clone() for t in (w.k8, w.v8, w.ks, w.vs)]

    q, k, v = (b.clone() for b in base)
    ops.lora_get_qkv(0, wl.x_qkv[0], q, k, v)
    q1 = w.cache.append(0, w.batch, k.view(T, -1, head_dim), v.view(T, -1, head_dim), q=q.view(T, -1, head_dim), rope=(table, pos))
    want = [q1.clone()] + [t.view(torch.uint8).clone() for t in (w.k8, w.v8, w.ks, w.vs)]
    for t, s0 in zip((w.k8, w.v8, w.ks, w.vs), start):
        t.view(torch.uint8).copy_(s0.view(torch.uint8))

    q, k, v = (b.clone() for b in base)
    ops.lora_get_qkv(0, wl.x_qkv[0], q, k, v, rope=(table, pos), kv_dest=(w.cache, w.batch), head_dim=head_dim)
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8)) for a, b in
               zip([q] + [t for t in (w.k8, w.v8, w.ks, w.vs)], want))
    q3 = q.view(T, -1, head_dim)
    lse = torch.empty(T, q3.size(1), device=DEV)
    o = w.cache.attend(0, w.batch, q3, lse=lse)
    _check_attend(w, q3, o, lse, None, None)
    out = torch.zeros(T, hidden, dtype=wl.dtype, device=DEV)
    ops.lora_get_o(0, o.view(T, -1), out)
    ops.plan.check()
    w.batch.check()
    assert out.abs().max() > 0
    # rotary alone, in place
    q, k, v = (b.clone() for b in base)
    ops.lora_get_qkv(0, wl.x_qkv[0], q, k, v, rope=(table, pos), head_dim=head_dim)
    assert torch.equal(q, want[0].view(T, -1))
    for bad in (dict(rope=(table, pos), kv_dest=(pos, k, v)), dict(rope=(table, pos[1:])), dict(rope=(sl.RotaryTable(256), pos))):
        with pytest.raises(RuntimeError):
            ops.lora_get_qkv(0, wl.x_qkv[0], q, k, v, head_dim=head_dim, **bad)


def test_a_refused_layer_changes_nothing():
    """``lora_get_qkv`` with a cache or a table that does not fit raises before it adds the deltas."""
    from slora_b200.workloads import build_workload
    sl = _sl()
    wl = build_workload(5, pool_rows=8192, n_adapters=12, decode_tokens=50, hidden=1024, h_kv=256).to(DEV)
    T = wl.T
    ops = sl.LoraBatchOps(wl.a_start, wl.a_len, wl.a_loc, wl.a_scaling, wl.pools_a, wl.pools_b, wl.max_rank)
    ops.prepare(wl.ids)
    g = torch.Generator().manual_seed(2)
    base = [torch.randn(T, n, generator=g).to(wl.dtype).to(DEV) for n in (1024, 256, 256)]
    table, pos = sl.RotaryTable(128), torch.arange(T, device=DEV)
    w = World([9] * T, [1] * T, 2, 128, 16, "int8")
    w.batch.q_start.copy_(torch.arange(T, dtype=torch.int32))
    other_heads = World([9] * T, [1] * T, 3, 128, 16, "int8").cache
    wide = torch.zeros(T, 1024 + 4, dtype=wl.dtype, device=DEV)
    cases = [dict(rope=(table, pos), kv_dest=(other_heads, w.batch)),           # the cache has other KV heads
             dict(rope=(table, pos.cpu()), kv_dest=(w.cache, w.batch)), dict(rope=(table, pos.cpu())),
             dict(rope=(table, pos.int())), dict(kv_dest=(other_heads, w.batch)),
             dict(rope=(table, pos), kv_dest=(w.cache, w.batch), q=wide[:, :1024]), dict(rope=(table, pos), q=wide[:, 4:])]
    cases.append(dict(rope=(table, pos), kv_dest=(sl.KvCache8(4, 16, 2, 128, layer_num=1), w.batch), layer=1))   # no such layer
    for case in cases:
        q, k, v = (b.clone() for b in base)
        if "q" in case:
            case["q"].copy_(q)
            q = case.pop("q")
        layer = case.pop("layer", 0)
        if layer and len(ops.key_buffer) <= layer:
            continue
        before = w.k8.view(torch.uint8).clone()
        with pytest.raises((RuntimeError, IndexError)):
            ops.lora_get_qkv(layer, wl.x_qkv[0], q, k, v, **case)
        torch.cuda.synchronize()
        assert torch.equal(q, base[0]) and torch.equal(k, base[1]) and torch.equal(v, base[2])
        assert torch.equal(w.k8.view(torch.uint8), before)
    q, k, v = (b.clone() for b in base)
    ops.lora_get_qkv(0, wl.x_qkv[0], q, k, v, rope=(table, pos), kv_dest=(w.cache, w.batch))
    assert not torch.equal(q, base[0]) and w.batch.status() == 0


def test_out_may_be_q_without_weights():
    w = World([700, 300, 40, 2000], [300, 5, 1, 1], 2, 128, 16, "int8")
    q = torch.randn(w.T, 8, 128, device=DEV).half()
    want = w.cache.attend(0, w.batch, q, out=q.clone())
    with pytest.raises(RuntimeError, match="overlaps"):
        w.cache.attend(0, w.batch, q, out=q, add_weights=True)
    assert w.cache.attend(0, w.batch, q, out=q) is q and torch.equal(q, want)


@pytest.mark.parametrize("new,io", [(1, "fp16"), (2, "bf16")])
def test_a_sequence_in_more_parts_than_the_join_holds_at_once(new, io):
    # 60000 keys of one KV head: every CTA has a part of them
    w = World([60000], [new], 1, 128, 128, "int8", track=False)
    _run_attend(w, 8, io)
    _run_attend(w, 8, io, window=50000)


@pytest.mark.parametrize("lens,new,hq,hkv,d,kind", [
    ([700, 5, 130], [1, 1, 1], 8, 2, 128, "int8"),
    ([700, 5, 130], [3, 2, 17], 8, 2, 64, "e4m3"),
    ([700, 5, 130], [1, 1, 1], 8, 2, 256, "int8"),
    ([700, 5, 130], [40, 2, 9], 8, 2, 256, "e4m3"),
])
@pytest.mark.parametrize("window", [0, 90])
def test_weights_with_scores_computed_again(lens, new, hq, hkv, d, kind, window):
    # a table for 2^24 tokens a sequence: scores of that many keys are not kept
    w = World(lens, new, hkv, d, 128, kind, max_pages=1 << 17)
    _run_attend(w, hq, "fp16", window=window, weights=True)


def test_calls_from_several_threads():
    import threading
    sl = _sl()
    page, results = [16, 32, 64, 128], {}

    def work(i):
        try:
            w = World([300 + 7 * i, 90], [1 + 60 * (i % 3), 5], 2, 64 * (1 + i % 2), page[i % 4], "int8", seed=i)
            d = w.d
            table, pos = sl.RotaryTable(d), torch.arange(w.T, device=DEV)
            g = torch.Generator().manual_seed(i)
            stream = torch.cuda.Stream()
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    q, x = (torch.randn(w.T, h, d, generator=g).half().to(DEV) for h in (8, 2))
                    q = w.cache.append(0, w.batch, x, x, q=q, rope=(table, pos))
                    out = w.cache.attend(0, w.batch, q, out=torch.zeros_like(q), add_weights=True)
                w.cache.evict(0, w.batch, 64, 8)
                stream.synchronize()
            results[i] = (w, q, out)
        except BaseException as e:      # shown by the main thread
            results[i] = e

    for run in range(2):
        threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for i in range(8):
            assert not isinstance(results[i], BaseException), results[i]
            assert results[i][0].batch.status() == 0
        if run == 0:
            first = {i: results[i][2].clone() for i in range(8)}
        else:
            assert all(torch.equal(first[i], results[i][2]) for i in range(8))


@pytest.mark.parametrize("hq,hkv,d,page,kind,io", [(32, 16, 128, 16, "int8", "bf16"), (64, 16, 64, 64, "e4m3", "fp16"),
                                                   (48, 16, 128, 128, "e4m3", "fp16"), (16, 16, 64, 32, "int8", "bf16")])
@pytest.mark.parametrize("window", [0, 100])
def test_chunks_of_a_batch_with_many_heads(hq, hkv, d, page, kind, io, window):
    # with this many (sequence, KV head) pairs the tensor-memory kernel takes sequences of 64 rows and more
    new = [64, 70, 1, 0, 130, 200, 33, 22, 300]
    lens = [64, 470, 300, 20, 129, 333, 900, 22, 1000]
    w = World(lens, new, hkv, d, page, kind)
    _run_attend(w, hq, io, window=window)
    # capacity for 2^24 tokens: the scores are not kept
    w = World(lens, new, hkv, d, page, kind, max_pages=(1 << 24) // page)
    _run_attend(w, hq, io, window=window, weights=True)


@pytest.mark.parametrize("lens,new,hq,hkv", [([1000], [400], 16, 1), ([2000, 700, 30], [100, 40, 30], 8, 2), ([9000], [1], 64, 1)])
def test_many_rows_of_few_heads(lens, new, hq, hkv):
    # few (sequence, KV head) pairs: the row kernel, its keys split over the GPU; the weights from kept scores
    for d in (64, 128):
        w = World(lens, new, hkv, d, 32, "int8")
        _run_attend(w, hq, "bf16")
        _run_attend(w, hq, "fp16", window=200, weights=True)


@pytest.mark.parametrize("lens,new,hq,hkv,max_pages", [
    ([300 + 11 * i for i in range(20)], [5] * 20, 64, 8, None),        # many heads: a warp goes through all row blocks
    ([1000], [400], 16, 1, None),                                      # many row blocks: shared by the warps of a CTA
    ([900, 300], [60, 9], 16, 2, 1 << 17),                             # scores computed again
])
def test_weights_repeat_whichever_way_they_are_added_up(lens, new, hq, hkv, max_pages):
    w = World(lens, new, hkv, 128, 128 if max_pages else 32, "int8", max_pages=max_pages)
    q = torch.randn(w.T, hq, 128, device=DEV, dtype=torch.bfloat16)
    before, first = w.w.clone(), None
    for _ in range(15):
        w.w.copy_(before)
        w.cache.attend(0, w.batch, q, add_weights=True)
        first = w.w.clone() if first is None else first
        assert torch.equal(w.w, first)
    w.w.copy_(before)
    _run_attend(w, hq, "bf16", weights=True)


def test_few_heads_have_the_whole_gpu():
    # one KV head: 64 rows took 25 times the time of 56 (one CTA walked the whole context), the weights of a chunk 15 times the
    # attention's
    def took(n, new, hq, weights):
        w = World([n], [new], 1, 128, 128, "int8")
        q = torch.randn(w.T, hq, 128, device=DEV).bfloat16()
        times = []
        for _ in range(12):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            w.cache.attend(0, w.batch, q, add_weights=weights)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return sorted(times)[len(times) // 2]

    assert took(32768, 1, 64, False) < 3 * took(32768, 1, 56, False)
    assert took(1000, 400, 16, True) < 6 * took(1000, 400, 16, False)
