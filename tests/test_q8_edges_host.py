"""Refusals and bookkeeping of the 8-bit cache that need no GPU, beside those of ``tests/test_q8_host.py``."""
import pytest

from jacq_b200 import _native, q8_cache

OK, NULL, RANGE = 0, 1, 3
FAKE = 1 << 20      # stands for a device pointer; never dereferenced on the host


@pytest.mark.parametrize("change,status", [
    (dict(batch=-1), RANGE), (dict(batch=65536), RANGE), (dict(width=-1), RANGE), (dict(rows=-1), RANGE), (dict(slots=0), NULL),
    (dict(tables=0), NULL), (dict(lens=0), NULL), (dict(out_tables=0), NULL), (dict(out_lens=0), NULL), (dict(batch=0), OK)])
def test_gather_refusals(native_lib, change, status):
    a = dict(tables=FAKE, width=8, lens=FAKE, by_slot=1, rows=4, slots=FAKE, batch=2, out_tables=FAKE, out_lens=FAKE)
    a.update(change)
    assert native_lib.kivi_b200_q8_gather_slots(*a.values(), 0) == status


@pytest.mark.parametrize("change,status", [
    (dict(batch=-1), RANGE), (dict(batch=65536), RANGE), (dict(rows=-1), RANGE), (dict(lens=0), NULL), (dict(slots=0), NULL),
    (dict(offsets=0), NULL), (dict(batch=0), OK), (dict(rows=0), OK)])
def test_advance_refusals(native_lib, change, status):
    a = dict(lens=FAKE, rows=4, slots=FAKE, offsets=FAKE, batch=2)
    a.update(change)
    assert native_lib.kivi_b200_q8_advance_slots(*a.values(), 0) == status


def test_wait_failures_reads_the_librarys_counter(native_lib, monkeypatch):
    class Fake:
        def kivi_b200_q8_wait_failures(self, out):
            out._obj.value = 3
            return self.status

    fake = Fake()
    monkeypatch.setattr(_native, "lib", lambda: fake)
    fake.status = 0
    assert q8_cache.wait_failures() == 3
    monkeypatch.setattr(_native, "check", lambda rc, where: (_ for _ in ()).throw(RuntimeError(where)) if rc else None)
    fake.status = 9
    with pytest.raises(RuntimeError, match="wait_failures"):
        q8_cache.wait_failures()
