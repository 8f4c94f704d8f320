"""8-bit KV cache and rotary positions, what needs no GPU: refusals before anything is launched, the frequencies of the
scalings, the cache's bookkeeping."""
import ctypes
import math
import os
import shutil
import subprocess

import pytest
import torch

import slora_b200 as sl
from slora_b200 import _lib
from tests.helpers import ROOT

FAKE = 0x1000      # 16-byte aligned, never read: checks come first
L = _lib.lib


def _cache(**kw):
    c = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, weights=FAKE, n_pages=10, page_tokens=16, kv_heads=2, head_dim=128,
             kind=0)
    c.update(kw)
    return _lib.Kv8Cache(*[c[n] for n, _ in _lib.Kv8Cache._fields_])


def _batch(**kw):
    b = dict(page_table=FAKE, table_stride=4, kv_len=FAKE, q_start=FAKE, q_len=FAKE, status=0, n_seq=2, max_pages=4,
             max_q_len=1)
    b.update(kw)
    return _lib.Kv8Batch(*[b[n] for n, _ in _lib.Kv8Batch._fields_])


def _append(c=None, b=None, **kw):
    a = dict(k=FAKE, v=FAKE, ks=256, vs=256, T=2, q=0, q_out=0, hq=0, qs=0, qos=0, pos=0, turns=0, rot=0, factor=1.0, layout=0,
             dtype=0)
    a.update(kw)
    return L.slora_kv8_append(ctypes.byref(c or _cache()), ctypes.byref(b or _batch()), *list(a.values())[:15], a["dtype"], 0)


def _attend(c=None, b=None, **kw):
    a = dict(q=FAKE, qs=512, T=2, hq=4, out=FAKE, os=512, lse=0, scale=1.0, window=0, add=0, ws=FAKE, wsb=1 << 30, dtype=0)
    a.update(kw)
    return L.slora_kv8_attend(ctypes.byref(c or _cache()), ctypes.byref(b or _batch()), *a.values(), 0)


def _evict(c=None, b=None, **kw):
    a = dict(budget=32, recent=8, sink=0, kept=FAKE, dest=FAKE, stride=4, pages=4)
    a.update(kw)
    return L.slora_kv8_evict(ctypes.byref(c or _cache()), ctypes.byref(b or _batch()), *a.values(), 0)


@pytest.mark.parametrize("bad,code", [
    (dict(k=0), -1), (dict(v_scale=0), -1), (dict(k=FAKE + 8), -2), (dict(kind=2), -3), (dict(page_tokens=24), -4),
    (dict(page_tokens=256), -4), (dict(page_tokens=0), -4), (dict(head_dim=96), -4), (dict(kv_heads=0), -4), (dict(n_pages=0), -4),
])
def test_cache_is_refused(bad, code):
    c = _cache(**bad)
    assert _append(c) == code and _attend(c) == code and _evict(c) == code
    assert L.slora_kv8_read(ctypes.byref(c), ctypes.byref(_batch()), 0, 4, FAKE, FAKE, 0, 0) == code
    assert L.slora_kv8_attend_workspace_bytes(ctypes.byref(c), ctypes.byref(_batch()), 2, 4, 0) == 0


@pytest.mark.parametrize("bad,code", [
    (dict(page_table=0), -1), (dict(kv_len=0), -1), (dict(q_len=0), -1), (dict(n_seq=-1), -4), (dict(max_q_len=-1), -4),
    (dict(table_stride=3), -4), (dict(max_pages=1 << 28, table_stride=1 << 28), -4), (dict(n_seq=(1 << 20) + 1), -4),
])
def test_batch_is_refused(bad, code):
    b = _batch(**bad)
    assert _append(b=b) == code and _attend(b=b) == code and _evict(b=b) == code


def test_append_is_refused():
    assert _append(dtype=5) == -3
    assert _append(k=0) == -1 and _append(v=0) == -1
    assert _append(k=FAKE + 4) == -2 and _append(vs=257) == -2
    assert _append(ks=248) == -4                                    # rows overlap
    assert _append(q=FAKE, q_out=FAKE, hq=4, qs=512, qos=512) == -1   # q without a table
    rope = dict(pos=FAKE, turns=FAKE, rot=128)
    assert _append(q=FAKE, q_out=0, hq=4, qs=512, qos=512, **rope) == -1
    assert _append(q=FAKE, q_out=FAKE, hq=0, qs=512, qos=512, **rope) == -4
    assert _append(**{**rope, "rot": 24}) == -4 and _append(**{**rope, "rot": 144}) == -4 and _append(**{**rope, "rot": 0}) == -4
    assert _append(**rope, layout=2) == -4 and _append(**{**rope, "pos": 0}) == -1
    assert _append(T=0) == 0 and _append(b=_batch(n_seq=0)) == 0 and _append(b=_batch(max_q_len=0)) == 0


def test_attend_is_refused():
    assert _attend(dtype=2) == -3
    assert _attend(hq=3) == -4 and _attend(hq=0) == -4
    assert _attend(q=0) == -1 and _attend(out=0) == -1 and _attend(q=FAKE + 2) == -2 and _attend(os=504) == -4
    assert _attend(window=-1) == -4
    assert _attend(_cache(weights=0), add=1) == -1
    assert _attend(ws=0) == -6 and _attend(wsb=64) == -6 and _attend(ws=FAKE + 4) == -2
    assert _attend(T=0) == 0 and _attend(b=_batch(n_seq=0)) == 0 and _attend(b=_batch(max_q_len=0)) == 0
    b, c = _batch(), _cache()
    plain = L.slora_kv8_attend_workspace_bytes(ctypes.byref(c), ctypes.byref(b), 2, 4, 0)
    more = L.slora_kv8_attend_workspace_bytes(ctypes.byref(c), ctypes.byref(b), 2, 4, 1)
    assert plain > 0 and more >= plain + 2 * 4 * 4


def test_rows_that_overlap_are_refused():
    # two tokens of four heads of 128.  What passes is stopped by the next check (no workspace, no k), so that nothing is launched
    rope = dict(pos=FAKE, turns=FAKE, rot=128, q=FAKE, hq=4, qs=512)

    def rotary(q_out, stride, q_stride):
        return L.slora_rotary(q_out, FAKE, FAKE, 0, 2, 4, 2, 128, 128, stride, 256, q_stride, 256, FAKE, FAKE, 1.0, 0, 0, 0, 0)

    for out, stride in ((FAKE + 16, 512), (FAKE + 512 * 2 - 16, 512), (FAKE, 520), (FAKE + 1024, 1024), (FAKE - 16, 512)):
        for rc in (_append(**rope, q_out=out, qos=stride), rotary(out, stride, 512), _attend(out=out, os=stride, add=1, ws=0)):
            assert rc == -4 and b"overlaps" in L.slora_last_error()
    assert _attend(add=1, out=FAKE, ws=0) == -4 and b"overlaps" in L.slora_last_error()     # the weights read q again
    assert _attend(out=FAKE, ws=0) == -6 and rotary(FAKE, 512, 512) == -1                   # in place
    for out in (FAKE + 1024, FAKE + 2048, FAKE - 1024, FAKE + 3 * 1024):                    # side by side in a wider buffer
        assert rotary(out, 2048, 2048) == -1 and _attend(qs=2048, out=out, os=2048, add=1, ws=0) == -6
    assert rotary(FAKE + 2 * 1024, 512, 512) == -1 and _attend(out=FAKE + 2 * 1024, add=1, ws=0) == -6   # one behind the other


def test_evict_is_refused():
    assert _evict(_cache(weights=0)) == -1 and _evict(kept=0) == -1 and _evict(dest=0) == -1
    assert _evict(budget=0) == -4 and _evict(recent=-1) == -4 and _evict(sink=-1) == -4 and _evict(recent=20, sink=20) == -4
    assert _evict(pages=1) == -4 and _evict(stride=3) == -4
    assert _evict(b=_batch(n_seq=0)) == 0
    # the selection counts a layer's weights in 32 bits
    assert _evict(_cache(n_pages=2 ** 31)) == -4 and _evict(_cache(n_pages=2 ** 62)) == -4


def test_a_layer_has_less_than_two_to_the_31_rows():
    # rows (tokens x heads) are counted in 32 bits: the largest cache passes these checks (no sequences: nothing is launched)
    none = _batch(n_seq=0)
    for n, page, heads in ((2 ** 26, 16, 2), (2 ** 31 // 128 // 3 + 1, 128, 3), (2 ** 15, 128, 512)):
        fits, over = _cache(n_pages=n - 1, page_tokens=page, kv_heads=heads), _cache(n_pages=n, page_tokens=page, kv_heads=heads)
        assert (n - 1) * page * heads < 2 ** 31 <= n * page * heads
        assert _append(fits, none) == 0 and _attend(fits, none, hq=heads) == 0 and _evict(fits, none) == 0
        assert _append(over, none) == -4 and _attend(over, none, hq=heads) == -4 and _evict(over, none) == -4


def test_read_is_refused():
    c, b = ctypes.byref(_cache()), ctypes.byref(_batch())
    assert L.slora_kv8_read(c, b, 0, 4, FAKE, FAKE, 9, 0) == -3
    assert L.slora_kv8_read(c, b, 0, 4, 0, FAKE, 0, 0) == -1
    assert L.slora_kv8_read(c, b, 0, 4, FAKE + 8, FAKE, 0, 0) == -2
    assert L.slora_kv8_read(c, b, 0, -1, FAKE, FAKE, 0, 0) == -4
    assert L.slora_kv8_read(c, b, 0, 0, FAKE, FAKE, 0, 0) == 0


def test_rotary_is_refused():
    def call(**kw):
        a = dict(qo=FAKE, ko=FAKE, q=FAKE, k=FAKE, T=4, hq=4, hk=2, d=128, rot=128, qos=512, kos=256, qs=512, ks=256, pos=FAKE,
                 turns=FAKE, factor=1.0, layout=0, inverse=0, dtype=0)
        a.update(kw)
        return L.slora_rotary(*a.values(), 0)
    assert call(dtype=3) == -3 and call(d=80) == -4 and call(rot=8) == -4 and call(rot=136) == -4 and call(layout=3) == -4
    assert call(T=-1) == -4 and call(hq=-1) == -4 and call(hk=70000) == -4
    assert call(q=0) == -1 and call(ko=0) == -1 and call(pos=0) == -1 and call(turns=0) == -1
    assert call(q=FAKE + 2) == -2 and call(qs=510) == -2 and call(kos=128) == -4
    assert call(T=0) == 0 and call(hq=0, hk=0) == 0


def test_python_refuses_cpu_tensors_and_wrong_shapes():
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        sl.KvBatch(torch.zeros(1, 1, dtype=torch.int64), *[torch.zeros(1, dtype=torch.int32)] * 3, 1)
    with pytest.raises(RuntimeError, match="kind"):
        sl.KvCache8(4, 16, 2, 64, kind="int4", device="cpu")
    with pytest.raises(RuntimeError, match="page_tokens=8"):
        sl.KvCache8(4, 8, 2, 64, device="cpu")
    with pytest.raises(RuntimeError, match="head_dim=80"):
        sl.KvCache8(4, 16, 2, 80, device="cpu")
    c = sl.KvCache8(4, 16, 2, 64, layer_num=2, track_weights=True, device="cpu")
    assert c.bytes_per_token() == 2 * (2 * 2 * (64 + 4 / 16) + 8)
    with pytest.raises(RuntimeError, match="one k, v"):
        sl.KvCache8.from_buffers(c.k, c.v[:1], c.k_scale, c.v_scale)
    with pytest.raises(RuntimeError, match="k_scale"):
        sl.KvCache8.from_buffers(c.k, c.v, [x.half() for x in c.k_scale], c.v_scale)
    with pytest.raises(RuntimeError, match="dtype"):
        sl.KvCache8.from_buffers([x.float() for x in c.k], c.v, c.k_scale, c.v_scale)
    got = c.pages.alloc(3)
    assert got.tolist() == [0, 1, 2] and c.pages.can_use_mem_size == 1
    c.pages.free(got[1:])
    assert c.pages.can_use_mem_size == 3
    with pytest.raises(Exception, match="enough"):
        c.pages.alloc(4)


def test_rotary_table_refuses():
    for kw, text in ((dict(head_dim=80), "head_dim"), (dict(head_dim=64, rotary_dim=24), "rotary_dim"),
                     (dict(head_dim=64, rotary_dim=0), "rotary_dim"), (dict(head_dim=64, layout="pairs"), "layout"),
                     (dict(head_dim=64, base=1.0), "base"), (dict(head_dim=64, scaling={"type": "what"}), "scaling"),
                     (dict(head_dim=64, scaling={"type": "linear"}), "needs 'factor'"),
                     (dict(head_dim=64, scaling={"type": "linear", "factor": 0.5}), "factor"),
                     (dict(head_dim=64, scaling={"type": "linear", "factor": 2.0, "beta_fast": 1.0}), "does not take"),
                     (dict(head_dim=64, scaling={"type": "llama3", "factor": 8.0, "low_freq_factor": 4.0, "high_freq_factor": 1.0,
                                                 "original_max_position": 8192}), "low_freq")):
        with pytest.raises(RuntimeError, match=text):
            sl.RotaryTable(device="cpu", **kw)


def test_rotary_frequencies():
    plain = sl.RotaryTable(64, device="cpu")
    assert plain.inv_freq[0] == 1.0 and math.isclose(plain.inv_freq[16], 10000.0 ** -0.5) and plain.factor == 1.0
    assert torch.allclose(plain.turns * 2 * math.pi, torch.tensor(plain.inv_freq, dtype=torch.float64), rtol=1e-15, atol=0)
    lin = sl.RotaryTable(64, scaling={"type": "linear", "factor": 4.0}, device="cpu")
    assert all(math.isclose(a, b / 4) for a, b in zip(lin.inv_freq, plain.inv_freq))
    ntk = sl.RotaryTable(64, scaling={"type": "ntk", "factor": 4.0}, device="cpu")      # fastest kept, slowest shrunk by 4
    assert ntk.inv_freq[0] == 1.0 and math.isclose(ntk.inv_freq[-1], plain.inv_freq[-1] / 4)
    yarn = sl.RotaryTable(64, scaling={"type": "yarn", "factor": 8.0, "original_max_position": 4096}, device="cpu")
    assert yarn.inv_freq[0] == 1.0 and math.isclose(yarn.inv_freq[-1], plain.inv_freq[-1] / 8)
    assert all(a / 8 <= b * (1 + 1e-12) and b <= a * (1 + 1e-12) for a, b in zip(plain.inv_freq, yarn.inv_freq))
    assert math.isclose(yarn.factor, 0.1 * math.log(8.0) + 1.0)
    l3 = sl.RotaryTable(128, base=500000.0, device="cpu", scaling={"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0,
                                                                  "high_freq_factor": 4.0, "original_max_position": 8192})
    base = sl.RotaryTable(128, base=500000.0, device="cpu")
    for a, b in zip(base.inv_freq, l3.inv_freq):
        wave = 2 * math.pi / a
        assert math.isclose(b, a) if wave < 2048 else math.isclose(b, a / 8) if wave > 8192 else a / 8 <= b <= a


def test_page_tables_whose_rows_overlap_are_refused():
    from slora_b200.kv_cache import _table_stride
    t = torch.arange(12).view(3, 4)
    assert _table_stride(t) == 4 and _table_stride(t[:, :2]) == 4 and _table_stride(t[:1].expand(1, 4)) == 4
    for bad in (t[:1].expand(3, 4), t.view(-1).as_strided((3, 4), (2, 1))):
        with pytest.raises(RuntimeError, match="overlap"):
            _table_stride(bad)
    with pytest.raises(RuntimeError, match="contiguous rows"):
        _table_stride(t.t())
    with pytest.raises(RuntimeError, match="contiguous rows"):
        _table_stride(t.int())


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_shared_memory_limit_of_two_threads(tmp_path):
    """Launches that ask for different sizes do not lower a kernel's limit for one another (tests/smem_limit_model.cpp)."""
    exe = str(tmp_path / "smem_limit")
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", os.path.join(ROOT, "slora_b200", "csrc"),
                    os.path.join(ROOT, "tests", "smem_limit_model.cpp"), "-o", exe], check=True)
    res = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0, res.stdout
