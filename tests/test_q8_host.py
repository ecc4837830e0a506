"""The 8-bit cache without a GPU: its oracle's own properties, byte accounting, and every refusal of the C entry
points, which check their arguments on the host before anything is launched."""
import ctypes

import pytest
import torch

from jacq_b200 import _native
from jacq_b200.q8_cache import Q8Cache, Q8Layout, evict_pages
from tests import q8_oracle as qo

OK, NULL, GEOM, RANGE, ALIGN, WORKSPACE, TABLE = 0, 1, 2, 3, 4, 5, 7
FAKE = 1 << 20      # stands for a device pointer; never dereferenced on the host


def geometry(nh=8, nkv=2, d=128, block=16, fmt=0):
    return _native.KiviQ8Geometry(nh, nkv, d, block, fmt)


def cache(**change):
    fields = dict(k_pages=FAKE, v_pages=FAKE, scales=FAKE, k_tail=FAKE, v_tail=FAKE, num_blocks=64, num_slots=4)
    fields.update(change)
    return _native.KiviQ8CacheStruct(*fields.values())


@pytest.mark.parametrize("bad", [dict(nh=7), dict(nkv=0), dict(nh=0), dict(d=96), dict(d=512), dict(d=0), dict(block=8),
                                 dict(block=48), dict(block=256), dict(fmt=2), dict(fmt=-1), dict(nh=32768)])
def test_geometry_is_refused(native_lib, bad):
    g = geometry(**bad)
    assert native_lib.kivi_b200_q8_validate_geometry(ctypes.byref(g)) == GEOM
    assert native_lib.kivi_b200_q8_attention_workspace_bytes(ctypes.byref(g), 1, 1, 100, 0, 0, 1) == 0


def test_geometry_is_accepted(native_lib):
    for d in (64, 128, 256):
        for block in (16, 32, 64, 128):
            for fmt in (0, 1):
                g = geometry(d=d, block=block, fmt=fmt)
                assert native_lib.kivi_b200_q8_validate_geometry(ctypes.byref(g)) == OK
    assert native_lib.kivi_b200_q8_validate_geometry(None) == NULL


def write_call(lib, g=None, c=None, **change):
    a = dict(new_k=FAKE, new_v=FAKE, ks=256, vs=256, tables=FAKE, width=8, starts=FAKE, offsets=FAKE, slots=0, batch=4,
             total=4, max_new=1, max_start=100)
    a.update(change)
    g, c = geometry() if g is None else g, cache() if c is None else c
    return lib.kivi_b200_q8_cache_write(ctypes.byref(g), ctypes.byref(c), *a.values(), 0)


@pytest.mark.parametrize("change,status", [
    (dict(new_k=0), NULL), (dict(new_v=0), NULL), (dict(tables=0), NULL), (dict(starts=0), NULL), (dict(offsets=0), NULL),
    (dict(new_k=FAKE + 8), ALIGN), (dict(ks=257), ALIGN), (dict(vs=260), ALIGN), (dict(ks=248), RANGE), (dict(vs=0), RANGE),
    (dict(batch=-1), RANGE), (dict(batch=5), RANGE), (dict(batch=65536, slots=FAKE), RANGE), (dict(width=-1), RANGE),
    (dict(total=-1), RANGE), (dict(max_new=-1), RANGE), (dict(max_start=-1), RANGE), (dict(max_new=1 << 30), RANGE),
    (dict(max_start=1 << 30), RANGE),
    (dict(batch=0), OK), (dict(total=0), OK), (dict(max_new=0), OK)])
def test_write_refusals(native_lib, change, status):
    assert write_call(native_lib, **change) == status


@pytest.mark.parametrize("change,status", [
    (dict(k_pages=0), NULL), (dict(v_pages=0), NULL), (dict(scales=0), NULL), (dict(k_tail=0), NULL), (dict(v_tail=0), NULL),
    (dict(k_pages=FAKE + 4), ALIGN), (dict(scales=FAKE + 8), ALIGN), (dict(v_tail=FAKE + 2), ALIGN), (dict(num_blocks=0), RANGE),
    (dict(num_slots=0), RANGE)])
def test_cache_refusals(native_lib, change, status):
    assert write_call(native_lib, c=cache(**change)) == status
    assert read_call(native_lib, c=cache(**change)) == status
    assert attend_call(native_lib, c=cache(**change)) == status


def read_call(lib, c=None, **change):
    a = dict(tables=FAKE, width=8, lens=FAKE, slots=0, offsets=FAKE, first=FAKE, batch=4, total=8, max_rows=4, k=FAKE, v=FAKE)
    a.update(change)
    g, c = geometry(), cache() if c is None else c
    return lib.kivi_b200_q8_cache_read(ctypes.byref(g), ctypes.byref(c), *a.values(), 0)


@pytest.mark.parametrize("change,status", [
    (dict(tables=0), NULL), (dict(lens=0), NULL), (dict(offsets=0), NULL), (dict(first=0), NULL), (dict(k=0), NULL),
    (dict(v=0), NULL), (dict(k=FAKE + 8), ALIGN), (dict(batch=5), RANGE), (dict(total=-1), RANGE), (dict(max_rows=-1), RANGE),
    (dict(batch=0), OK), (dict(total=0), OK), (dict(max_rows=0), OK)])
def test_read_refusals(native_lib, change, status):
    assert read_call(native_lib, **change) == status


def attend_call(lib, g=None, c=None, **change):
    a = dict(q=FAKE, stride=1024, offsets=0, total=4, tables=FAKE, width=8, lens=FAKE, slots=0, batch=4, max_q=1, max_len=128,
             window=0, sinks=0, scale=0.0, mass=0, mass_width=0, out32=FAKE, out16=0, ws=0, ws_bytes=0)
    a.update(change)
    g, c = geometry() if g is None else g, cache() if c is None else c
    return lib.kivi_b200_q8_attention(ctypes.byref(g), ctypes.byref(c), *a.values(), 0)


@pytest.mark.parametrize("change,status", [
    (dict(q=0), NULL), (dict(tables=0), NULL), (dict(lens=0), NULL), (dict(out32=0), NULL), (dict(out16=FAKE), RANGE),
    (dict(q=FAKE + 2), ALIGN), (dict(stride=1025), ALIGN), (dict(out32=FAKE + 4), ALIGN), (dict(stride=1016), RANGE),
    (dict(batch=5, total=5), RANGE), (dict(total=3), RANGE), (dict(max_q=2), RANGE), (dict(max_len=-1), RANGE),
    (dict(max_len=1 << 30), RANGE), (dict(window=-1), RANGE), (dict(sinks=-1), RANGE), (dict(scale=-1.0), RANGE),
    (dict(scale=float("nan")), RANGE), (dict(scale=float("inf")), RANGE), (dict(max_len=144), TABLE),
    (dict(offsets=FAKE, total=1 << 28, max_q=1 << 28), RANGE),
    (dict(mass=FAKE, mass_width=7), RANGE), (dict(mass=FAKE, mass_width=8), WORKSPACE),
    (dict(mass=FAKE, mass_width=8, ws=FAKE, ws_bytes=16), WORKSPACE), (dict(mass=FAKE, mass_width=8, ws=FAKE + 8, ws_bytes=1 << 20), ALIGN),
    (dict(mass=FAKE, mass_width=8, ws=FAKE, ws_bytes=1 << 20, offsets=FAKE), RANGE),
    (dict(batch=0, total=0), OK), (dict(offsets=FAKE, total=0), OK), (dict(offsets=FAKE, max_q=0), OK)])
def test_attention_refusals(native_lib, change, status):
    assert attend_call(native_lib, **change) == status


def evict_call(lib, **change):
    a = dict(nkv=2, block=16, tables=FAKE, width=8, lens=FAKE + 1, mass=FAKE, mass_width=8, batch=2, max_len=128, budget=4, first=1,
             recent=2, new_tables=FAKE + 64, new_lens=FAKE + 128, new_mass=FAKE + 192, freed=FAKE + 256, counts=FAKE + 320)
    a.update(change)
    return lib.kivi_b200_q8_evict(*a.values(), 0)


@pytest.mark.parametrize("change,status", [
    (dict(nkv=0), GEOM), (dict(block=24), GEOM), (dict(tables=0), NULL), (dict(lens=0), NULL), (dict(mass=0), NULL),
    (dict(new_tables=0), NULL), (dict(new_lens=0), NULL), (dict(new_mass=0), NULL), (dict(freed=0), NULL), (dict(counts=0), NULL),
    (dict(batch=-1), RANGE), (dict(width=0), RANGE), (dict(mass_width=7), RANGE), (dict(max_len=-1), RANGE), (dict(budget=-1), RANGE),
    (dict(first=3), RANGE), (dict(first=-1), RANGE), (dict(recent=-1), RANGE), (dict(recent=4), RANGE), (dict(max_len=144, mass_width=9), TABLE),
    (dict(new_tables=FAKE), RANGE), (dict(new_mass=FAKE), RANGE), (dict(freed=FAKE), RANGE), (dict(freed=FAKE + 64), RANGE),
    (dict(width=1 << 20), RANGE), (dict(batch=0), OK)])
def test_evict_refusals(native_lib, change, status):
    assert evict_call(native_lib, **change) == status


def test_rejected_count_needs_a_place(native_lib):
    assert native_lib.kivi_b200_q8_rejected_indices(None) == NULL


def test_layout_refusals_and_cpu_tensors():
    for bad in (Q8Layout(7, 2, 128), Q8Layout(8, 2, 96), Q8Layout(8, 2, 128, 8), Q8Layout(8, 2, 128, 16, "fp4"), Q8Layout(8, 0, 128)):
        with pytest.raises(ValueError):
            bad.validate()
    with pytest.raises(RuntimeError, match="CUDA"):
        Q8Cache(Q8Layout(8, 2, 128), 4, 1, 4, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        evict_pages(torch.zeros((1, 4), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros((1, 2, 4)), block_size=16,
                    budget=1, max_seq_len=10)


def test_bytes_of_a_decode_step():
    lay = Q8Layout(32, 8, 128, 16)
    assert lay.page_bytes() == 8 * (2 * 16 * 128 + 8)
    # 8192 tokens: 512 pages, no tail; q in fp16, out in fp16
    assert lay.decode_algorithmic_bytes(8192) == 8 * 128 * 2 * 8192 + 512 * 68 + 4 * 32 * 128
    # 5 tail rows in fp16
    assert lay.decode_algorithmic_bytes(21) == 8 * 128 * (2 * 16 + 4 * 5) + 68 + 4 * 32 * 128
    assert lay.decode_algorithmic_bytes(8192, window=16, sinks=16) == 8 * 128 * 64 + 2 * 68 + 4 * 32 * 128
    assert lay.decode_algorithmic_bytes(0) == 4 * 32 * 128


def test_workspace_bytes_follow_the_visible_context(native_lib):
    g = geometry()
    ask = lambda *a: native_lib.kivi_b200_q8_attention_workspace_bytes(ctypes.byref(g), *a)  # noqa: E731
    assert ask(400, 1, 512, 0, 0, 0) == 0           # units enough to fill the GPU uncut: nothing to join
    full, windowed = ask(4, 1, 4096, 0, 0, 1), ask(4, 1, 4096, 256, 4, 1)
    assert full >= 4 * 2 * 256 * 8 * 8 and 0 < windowed < full // 8
    for bad in ((0, 1, 10, 0, 0, 1), (1, 0, 10, 0, 0, 1), (1, 1, -1, 0, 0, 1), (1, 1, 10, -1, 0, 1), (1, 1, 10, 0, -1, 1)):
        assert ask(*bad) == 0


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_oracle_rounds_by_at_most_half_a_step(fmt):
    gen = torch.Generator().manual_seed(3)
    x = (torch.randn((64, 32), generator=gen) * torch.exp(torch.randn((64, 1), generator=gen) * 3)).half()
    codes, scale = qo.quantise(x, fmt)
    err = (qo.dequantise(codes, scale) - x.double()).abs()
    if fmt == "int8":   # half a code, and the fp32 rounding of the scale and the quotient
        assert float(err.max()) <= float(scale) * (0.5 + 128 * 2.0 ** -23)
    else:               # half of e4m3's step at the value: 2^-4 relative, or half the subnormal step 2^-9
        assert (err <= torch.maximum(x.double().abs() * 2.0 ** -4, torch.tensor(float(scale) * 2.0 ** -10)) * (1 + 2.0 ** -20)).all()
    assert int(qo.quantise(torch.zeros(16, 8).half(), fmt)[0].float().abs().max()) == 0
    assert qo.quantise(torch.full((16, 8), float("inf")).half(), fmt)[1].isnan()


def test_oracle_eviction_orders_ties_nan_and_protected_pages():
    mass = torch.tensor([[5.0, 1.0, 1.0, float("nan"), 3.0, 0.0, 9.0, 2.0]])
    assert qo.evict(8, mass, 8, 0, 0) == list(range(8))
    assert qo.evict(8, mass, 3, 0, 0) == [0, 4, 6]
    assert qo.evict(8, mass, 5, 0, 0) == [0, 1, 4, 6, 7]        # 1 before 2: the lower index of a tie
    assert qo.evict(8, mass, 7, 0, 0) == [0, 1, 2, 4, 5, 6, 7]  # NaN goes first
    assert qo.evict(8, mass, 3, 1, 2) == [0, 6, 7]
    assert qo.evict(8, mass, 0, 0, 0) == []
