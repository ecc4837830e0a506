"""The 8-bit cache on the GPU against the plain oracle in 64 bits (``tests/q8_oracle.py``): writer and read-back bit for
bit, attention within bounds derived from its roundings, masses, evictions exactly; then all of it as it is used."""
import random

import pytest
import torch

from jacq_b200.q8_cache import Q8Cache, Q8CacheTensors, Q8Layout, evict_pages, rejected_indices
from tests import q8_oracle as qo

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HALF = 2.0 ** -11    # half a step of fp16, relative


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def offsets_of(counts):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return at


class World:
    """A cache of its own, the fp16 rows every sequence was fed, and scattered pages and slots."""

    def __init__(self, layout, capacity, seed=0, spare=3, slots=None):
        self.layout, self.gen, rng = layout, torch.Generator().manual_seed(seed), random.Random(seed)
        n, b = len(capacity), layout.block_size
        width = max(1, max(-(-c // b) for c in capacity))
        need = [c // b for c in capacity]
        pool = list(range(sum(need) + spare))
        rng.shuffle(pool)
        self.n, self.slots = n, slots
        count = n if slots is None else max(slots) + 1
        self.cache = Q8Cache(layout, len(pool), count, width, DEV)
        tables, at = torch.zeros((count, width), dtype=torch.int32), 0
        for i in range(n):
            row = i if slots is None else slots[i]
            tables[row, :need[i]] = torch.tensor(pool[at:at + need[i]], dtype=torch.int32)
            at += need[i]
        self.free = pool[at:]
        self.cache.set_block_tables(tables)
        self.rows = [(torch.zeros((0, layout.num_kv_heads, layout.head_dim), dtype=torch.float16),) * 2 for _ in range(n)]

    def randn(self, *shape, k=False):
        x = torch.randn(shape, generator=self.gen)
        if k:
            x[..., 1::29] *= 10.0
        return x.half()

    def feed(self, counts, k=None, v=None, max_new=None):
        nkv, d = self.layout.num_kv_heads, self.layout.head_dim
        total = sum(counts)
        k = self.randn(total, nkv, d, k=True) if k is None else k
        v = self.randn(total, nkv, d) if v is None else v
        at = offsets_of(counts)
        self.cache.write(k.to(DEV), v.to(DEV), i32(at), max_new_per_seq=max_new or max(counts),
                         max_start_seq_len=max(r[0].shape[0] for r in self.rows),
                         slot_ids=None if self.slots is None else i32(self.slots))
        for i in range(self.n):
            self.rows[i] = tuple(torch.cat([old, new[at[i]:at[i + 1]]]) for old, new in zip(self.rows[i], (k, v)))

    def lens(self):
        return [r[0].shape[0] for r in self.rows]

    def held(self):
        """Per sequence the K and V the cache stands for, in 64 bits."""
        return [tuple(qo.cached(x, self.layout.block_size, self.layout.fmt) for x in r) for r in self.rows]

    def check_contents(self):
        lay, c = self.layout, self.cache
        b = lay.block_size
        for i, r in enumerate(self.rows):
            slot = i if self.slots is None else self.slots[i]
            t = r[0].shape[0]
            assert int(c.seq_lens[slot]) == t
            for which, (rows, pages, tail) in enumerate(zip(r, (c.tensors.K_PAGES, c.tensors.V_PAGES), (c.tensors.K_TAIL, c.tensors.V_TAIL))):
                ids = c.block_tables[slot, :t // b].long()
                codes = pages.view(torch.int8)[ids].cpu()
                scales = c.tensors.SCALES[ids, :, which].cpu()
                for p in range(t // b):
                    for h in range(lay.num_kv_heads):
                        want, scale = qo.quantise(rows[p * b:(p + 1) * b, h], lay.fmt)
                        got = scales[p, h]
                        assert torch.equal(got, scale) or (got.isnan() and scale.isnan()), (i, which, p, h, float(got), float(scale))
                        assert torch.equal(codes[p, h], want.view(torch.int8)), (i, which, p, h)
                live = rows[t // b * b:].transpose(0, 1)
                assert torch.equal(tail[slot, :, :t % b].cpu().view(torch.int16), live.contiguous().view(torch.int16)), (i, which)

    def attend(self, q, counts=None, half=True, **kw):
        out = torch.full(q.shape, 7.0, dtype=torch.float16 if half else torch.float32, device=DEV)
        kw.setdefault("max_seq_len", max(self.lens()))
        if counts is not None:
            kw.update(q_offsets=i32(offsets_of(counts)), max_q_per_seq=max(counts))
        self.cache.attend(q.to(DEV), out, slot_ids=None if self.slots is None else i32(self.slots), **kw)
        return out.cpu().double()

    def check_attention(self, counts=None, half=True, window=0, sinks=0, scale=None, held=None, **kw):
        """Attention of each sequence's last tokens within the oracle's bound; returns the weights per sequence."""
        lay = self.layout
        n = [1] * self.n if counts is None else counts
        q = self.randn(sum(n), lay.num_q_heads, lay.head_dim)
        got = self.attend(q, counts, half, window=window, sinks=sinks, scale=scale, **kw)
        at, all_weights = offsets_of(n), []
        for i, (k, v) in enumerate(self.held() if held is None else held):
            want, weights, bound = qo.attend(q[at[i]:at[i + 1]], k, v, window, sinks, scale)
            if half:   # the output's own rounding: half a step, or half a subnormal one
                bound = bound + HALF * want.abs() + 2.0 ** -25
            err = (got[at[i]:at[i + 1]] - want).abs()
            assert torch.isfinite(got[at[i]:at[i + 1]]).all() and (err <= bound).all(), \
                (i, float((err - bound).max()), float(err.max()), (err > bound).nonzero()[:3].tolist())
            all_weights.append(weights)
        return all_weights


LAYOUTS = [Q8Layout(8, 2, 128, 16, "int8"), Q8Layout(3, 3, 64, 32, "e4m3"), Q8Layout(14, 2, 64, 16, "int8"), Q8Layout(10, 1, 128, 64, "e4m3"),
           Q8Layout(4, 2, 256, 128, "int8"), Q8Layout(16, 1, 256, 16, "e4m3"), Q8Layout(24, 1, 64, 16, "int8"), Q8Layout(5, 5, 128, 32, "int8")]
IDS = [f"{x.num_q_heads}/{x.num_kv_heads}x{x.head_dim}b{x.block_size}{x.fmt}" for x in LAYOUTS]


# ------------------------------------------------------------------------------------------------ writer and read-back

@pytest.mark.parametrize("layout", LAYOUTS, ids=IDS)
def test_writer_is_bit_exact(layout, native_lib):
    b = layout.block_size
    w = World(layout, [6 * b + 5] * 6, seed=1)
    before = rejected_indices()
    w.feed([0, 1, b - 1, b, b + 1, 3 * b + 7])
    w.check_contents()
    w.feed([1, b - 1, 1, 2 * b, 0, b])       # completes open blocks, leaves one sequence alone
    w.check_contents()
    w.feed([2 * b + 3, 1, 5, 1, b - 2, 1])
    w.check_contents()
    torch.cuda.synchronize()
    assert rejected_indices() == before
    # pages that no table names, and tail rows behind the last token, stay as they were
    free = torch.tensor(w.free, device=DEV)
    assert int(w.cache.tensors.K_PAGES.view(torch.int8)[free].abs().max()) == 0
    t = w.lens()[0]
    assert int(w.cache.tensors.K_TAIL[0, :, max(t % b, 1):].abs().max() if t >= b and t % b < 1 else 0) == 0


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_a_chunk_equals_its_tokens(fmt, native_lib):
    layout = Q8Layout(4, 2, 128, 16, fmt)
    a, b = World(layout, [70, 70], seed=2), World(layout, [70, 70], seed=2)
    k, v = a.randn(70, 2, 128, k=True), a.randn(70, 2, 128)
    a.feed([37, 33], k, v)
    for t in range(37):
        counts = [1, 1 if t < 33 else 0]
        rows = [t] + ([37 + t] if t < 33 else [])
        b.feed(counts, k[rows], v[rows])
    for x, y in list(zip(a.cache.tensors, b.cache.tensors))[:3]:      # tail rows behind the last token may differ
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    a.check_contents()
    b.check_contents()


def test_writer_takes_strided_slices_and_slots(native_lib):
    layout = Q8Layout(8, 2, 64, 16, "int8")
    w = World(layout, [60, 60, 60], seed=3, slots=[4, 0, 2])
    counts, total = [17, 40, 3], 60
    fused = w.randn(total, (8 + 4) * 64).to(DEV)
    k, v = fused[:, 8 * 64:10 * 64].view(total, 2, 64), fused[:, 10 * 64:].view(total, 2, 64)
    w.cache.write(k, v, i32(offsets_of(counts)), max_new_per_seq=40, max_start_seq_len=0, slot_ids=i32(w.slots))
    at = offsets_of(counts)
    w.rows = [(k[at[i]:at[i + 1]].cpu(), v[at[i]:at[i + 1]].cpu()) for i in range(3)]
    w.check_contents()
    assert w.cache.seq_lens.tolist() == [40, 0, 3, 0, 17]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_writer_extremes(fmt, native_lib):
    """All-zero blocks, the smallest and largest fp16 values, and blocks with an infinity or a NaN."""
    layout = Q8Layout(2, 2, 64, 16, fmt)
    w = World(layout, [100], seed=4)
    k, v = w.randn(100, 2, 64, k=True), w.randn(100, 2, 64)
    k[:16] = 0.0
    k[16:32] = torch.where(torch.rand((16, 2, 64), generator=w.gen) < 0.5, 2.0 ** -24, -(2.0 ** -24)).half()
    k[32:48] *= 6000.0
    k[40, 0, 3] = 65504.0
    k[50, 1, 7] = float("inf")
    k[70, 0, 0] = float("nan")
    v[80, 1, 63] = float("-inf")
    v[95:] = -0.0
    w.feed([100], k, v)
    w.check_contents()


@pytest.mark.parametrize("layout", LAYOUTS[:5], ids=IDS[:5])
def test_read_back(layout, native_lib):
    b = layout.block_size
    w = World(layout, [4 * b + 9] * 4, seed=5)
    w.feed([4 * b + 3, b, 7, 1])
    first, rows = [b - 5, 0, 3, 0], [2 * b + 9, b, 4, 1]
    k, v = w.cache.read(i32(offsets_of(rows)), i32(first), total=sum(rows), max_rows_per_seq=max(rows))
    at = offsets_of(rows)
    for i, held in enumerate(w.held()):
        for got, x in zip((k, v), held):
            got = got[at[i]:at[i + 1]].cpu()
            want = x[first[i]:first[i] + rows[i]].float().half()    # code * scale in fp32, then fp16
            paged = max(0, min(rows[i], w.lens()[i] // b * b - first[i]))
            assert torch.equal(got[paged:], want[paged:])
            assert ((got[:paged].double() - x[first[i]:first[i] + paged]).abs() <= HALF * (1 + 2.0 ** -12) * x[first[i]:first[i] + paged].abs() + 2.0 ** -25).all()
    # rows behind the last token are zeros
    k, v = w.cache.read(i32([0, 0, 0, 12, 12]), i32([0, 0, 3, 0]), total=12, max_rows_per_seq=12)
    assert torch.equal(k[:4].cpu(), w.rows[2][0][3:]) and int(k[4:].abs().max()) == 0 and int(v[4:].abs().max()) == 0


# ------------------------------------------------------------------------------------------------ attention

@pytest.mark.parametrize("layout", LAYOUTS, ids=IDS)
def test_attention_of_single_tokens(layout, native_lib):
    b = layout.block_size
    lens = [1, 15, 16, 17, b, b + 1, 2 * b - 1, 5 * b + 3, 600, 333]
    w = World(layout, lens, seed=6)
    w.feed(lens)
    for half in (True, False):
        w.check_attention(half=half)
    w.check_attention(scale=0.3)
    for window, sinks in ((1, 0), (5, 1), (16, 4), (100, 17), (100, 1000), (333, 0), (1000, 4), (2 * b, 3 * b)):
        w.check_attention(window=window, sinks=sinks)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_attention_of_empty_and_unequal_sequences(fmt, native_lib):
    layout = Q8Layout(8, 4, 64, 16, fmt)
    w = World(layout, [0, 40, 0, 2000, 1], seed=7)
    w.feed([0, 40, 0, 2000, 1])
    q = w.randn(5, 8, 64)
    got = w.attend(q, half=True)
    assert int(got[0].abs().max()) == 0 and int(got[2].abs().max()) == 0     # nothing to see: zeros
    w.check_attention(max_seq_len=2000)
    w.check_attention(max_seq_len=2015)    # a looser bound changes nothing but the launch


def test_a_cache_without_a_page(native_lib):
    """Nothing written yet, or fewer tokens than a page: tables may have no entry at all."""
    layout = Q8Layout(4, 2, 64, 128, "int8")
    w = World(layout, [0, 0], seed=23)
    w.cache = Q8Cache(layout, 1, 2, 0, DEV)
    assert int(w.attend(w.randn(2, 4, 64), max_seq_len=0).abs().max()) == 0
    mass = torch.zeros((2, 2, 1), device=DEV)
    w.attend(w.randn(2, 4, 64), max_seq_len=0, page_mass=mass)
    assert int(mass.abs().max()) == 0
    w.feed([5, 100])
    w.check_attention()
    w.check_attention([5, 40], window=3)


@pytest.mark.parametrize("layout", LAYOUTS, ids=IDS)
def test_attention_of_runs_of_tokens(layout, native_lib):
    b = layout.block_size
    lens, counts = [1, 9, b + 5, 3 * b, 400], [1, 9, 3, b + 2, 33]
    counts = [min(c, t) for c, t in zip(counts, lens)]
    w = World(layout, lens, seed=8)
    w.feed(lens)
    w.check_attention(counts)
    w.check_attention(counts, half=False, window=7, sinks=2)
    w.check_attention(counts, window=b + 3, sinks=20)
    w.check_attention([0, 1, 0, 2, 40], window=50)


def test_a_run_longer_than_its_sequence_gives_zeros_for_tokens_before_the_first(native_lib):
    layout = Q8Layout(4, 2, 128, 16, "int8")
    w = World(layout, [20], seed=9)
    w.feed([20])
    q = w.randn(24, 4, 128)
    got = w.attend(q, [24])
    assert int(got[:4].abs().max()) == 0
    held = w.held()[0]
    want, _, bound = qo.attend(q[4:], *held)
    assert ((got[4:] - want).abs() <= bound + HALF * want.abs() + 2.0 ** -25).all()


def test_attention_with_strided_queries(native_lib):
    layout = Q8Layout(8, 2, 64, 16, "int8")
    w = World(layout, [100, 30], seed=10)
    w.feed([100, 30])
    fused = w.randn(2, (8 + 4) * 64).to(DEV)
    q = fused[:, :8 * 64].view(2, 8, 64)
    got = w.cache.attend(q, max_seq_len=100).cpu()
    assert torch.equal(got, w.cache.attend(q.contiguous(), max_seq_len=100).cpu())


@pytest.mark.parametrize("layout", [LAYOUTS[0], LAYOUTS[1], LAYOUTS[4]], ids=["int8", "e4m3", "int8b128"])
def test_masked_infinities_and_nan_do_not_reach_a_row(layout, native_lib):
    """Tokens outside the window, before or after it, in a page or in the tail, may hold anything."""
    b = layout.block_size
    lens = [6 * b + 7, 6 * b + 7]
    w = World(layout, lens, seed=11)
    k, v = w.randn(sum(lens), layout.num_kv_heads, layout.head_dim, k=True), w.randn(sum(lens), layout.num_kv_heads, layout.head_dim)
    for x in (k, v):
        x[b + 3, :, 5] = float("nan")            # page 1 of sequence 0: its whole page is poisoned
        x[2 * b + 1, 0, 0] = float("inf")        # page 2, one head
        x[lens[0] + 4 * b, :, :] = float("-inf")  # page 4 of sequence 1
    w.feed(lens, k, v)
    w.check_contents()
    held = [(w.held()[0][0].nan_to_num(), w.held()[0][1].nan_to_num()), (w.held()[1][0].nan_to_num(), w.held()[1][1].nan_to_num())]
    # windows that leave pages 1, 2 (and 4) out, and first tokens of page 0 in
    w.check_attention(window=b + 7, sinks=min(b, 20), held=held)
    w.check_attention([5, 5], window=b + 2, sinks=1, held=held)
    # seen: the row is NaN, in that head alone
    got = w.attend(w.randn(2, layout.num_q_heads, layout.head_dim), window=5 * b + 6, sinks=0)
    assert got[0].isnan().all() and got[1].isnan().all()
    got = w.attend(w.randn(2, layout.num_q_heads, layout.head_dim), window=4 * b + 6, sinks=0)
    per = layout.num_q_heads // layout.num_kv_heads
    assert got[0, :per].isnan().all() and got[0, per:].isfinite().all()


def test_non_finite_tail_rows_reach_only_the_rows_that_see_them(native_lib):
    layout = Q8Layout(4, 2, 128, 32, "int8")
    w = World(layout, [60], seed=12)
    k, v = w.randn(60, 2, 128, k=True), w.randn(60, 2, 128)
    v[50, 0, 9] = float("inf")
    v[56, 1, 100] = float("nan")
    w.feed([60], k, v)
    q = w.randn(14, 4, 128)                      # tokens 46 .. 59
    got = w.attend(q, [14])
    clean = [x.clone() for x in w.held()[0]]
    clean[1][50, 0, 9] = 0.0
    clean[1][56, 1, 100] = 0.0
    want, _, bound = qo.attend(q, *clean)
    fine = (got - want).abs() <= bound + HALF * want.abs() + 2.0 ** -25
    hit = torch.zeros_like(fine)
    hit[4:, :2, 9] = True                        # token 50 on, heads of kv head 0
    hit[10:, 2:, 100] = True                     # token 56 on, heads of kv head 1
    assert fine[~hit].all() and got[hit].isnan().all()


def test_garbage_behind_the_last_token_is_never_read(native_lib):
    layout = Q8Layout(8, 2, 64, 16, "e4m3")
    w = World(layout, [37, 16, 5], seed=13)
    w.feed([37, 16, 5])
    for tail in (w.cache.tensors.K_TAIL, w.cache.tensors.V_TAIL):
        for i, t in enumerate((37, 16, 5)):
            tail[i, :, t % 16:] = float("nan")
    free = torch.tensor(w.free, device=DEV)
    w.cache.tensors.V_PAGES.view(torch.uint8)[free] = 0x7f     # NaN codes in pages that no table names
    w.cache.tensors.SCALES[free] = float("nan")
    w.check_attention()
    w.check_attention(window=9, sinks=1)
    w.check_attention([5, 2, 5])


def test_peaked_scores_and_very_unequal_scales(native_lib):
    """Softmax far from flat, and pages whose V scales differ by 2^16 in either order."""
    layout = Q8Layout(4, 1, 128, 16, "int8")
    for order in (1, -1):
        w = World(layout, [160], seed=14)
        k, v = w.randn(160, 1, 128, k=True), w.randn(160, 1, 128)
        scale = 2.0 ** (order * torch.linspace(-8, 8, 10))
        v = (v.float() * scale.repeat_interleave(16)[:, None, None]).half()
        k[3] = 8.0
        k[77] = -8.0
        w.feed([160], k, v)
        w.check_attention(scale=1.0)
        w.check_attention(scale=0.01)


def test_pages_beyond_four_gigabytes(native_lib):
    layout = Q8Layout(8, 8, 128, 16, "int8")
    page = 8 * 16 * 128
    blocks = (1 << 32) // page + 40
    w = World(layout, [100, 64], seed=15)
    w.cache = Q8Cache(layout, blocks, 2, w.cache.max_blocks_per_seq, DEV)
    tables = torch.tensor([[blocks - 1 - 2 * i for i in range(6)], [blocks - 2 - 2 * i for i in range(4)] + [0, 0]], dtype=torch.int32)
    w.cache.set_block_tables(torch.nn.functional.pad(tables, (0, w.cache.max_blocks_per_seq - 6)))
    w.feed([100, 64])
    w.check_contents()
    w.check_attention()
    k, _ = w.cache.read(i32([0, 100, 164]), i32([0, 0]), total=164, max_rows_per_seq=100)
    assert ((k[:100].cpu().double() - w.held()[0][0]).abs() <= HALF * 1.001 * w.held()[0][0].abs() + 2.0 ** -25).all()


class Large:
    """A batch too large for the oracle's loops: codes quantised by the library's own writer (whose bits the tests above
    pin) and read back, attention against the oracle in 64 bits on the device."""

    def __init__(self, layout, lens, seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.layout, self.lens, self.g = layout, lens, g
        nkv, b, d = layout.num_kv_heads, layout.block_size, layout.head_dim
        width = max(1, -(-max(lens) // b))
        self.cache = Q8Cache(layout, len(lens) * width + 1, len(lens), width, DEV)
        ids = torch.randperm(len(lens) * width, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        self.cache.set_block_tables(ids.view(len(lens), width))
        total = sum(lens)
        self.k, self.v = (torch.randn((total, nkv, d), generator=g, device=DEV).half() for _ in range(2))
        self.k[..., 1::29] *= 10.0
        self.at = offsets_of(lens)
        self.cache.write(self.k, self.v, i32(self.at), max_new_per_seq=max(lens), max_start_seq_len=0)
        self.scales = [float(x) for x in self.cache.tensors.SCALES.nan_to_num().amax((0, 1))]

    def held(self, i):
        """K and V of sequence i in 64 bits: the pages' codes times their scales, the tail as it is."""
        t, c = self.lens[i], self.cache
        b, nkv, d = self.layout.block_size, self.layout.num_kv_heads, self.layout.head_dim
        ids, got = c.block_tables[i, :t // b].long(), []
        for j, (pages, rows) in enumerate(((c.tensors.K_PAGES, self.k), (c.tensors.V_PAGES, self.v))):
            codes = pages.view(torch.int8)[ids].view(pages.dtype).float().double()
            x = (codes * c.tensors.SCALES[ids, :, j].double()[..., None, None]).transpose(1, 2).reshape(-1, nkv, d)
            got.append(torch.cat([x, rows[self.at[i] + t // b * b:self.at[i + 1]].double()]))
        return got

    def check(self, counts, window=0, sinks=0, half=True, products=2):
        lay = self.layout
        q = torch.randn((sum(counts), lay.num_q_heads, lay.head_dim), generator=self.g, device=DEV).half()
        got = torch.full(q.shape, 9.0, dtype=torch.float16 if half else torch.float32, device=DEV)
        kw = {} if max(counts) == 1 and min(counts) == 1 else dict(q_offsets=i32(offsets_of(counts)), max_q_per_seq=max(counts))
        self.cache.attend(q, got, max_seq_len=max(self.lens), window=window, sinks=sinks, **kw)
        at = offsets_of(counts)
        for i, n in enumerate(counts):
            if not n:
                continue
            bias = 128.0 * self.scales[0] if products == 1 and lay.fmt == "int8" else 0.0
            want, bound = qo.attend_block(q[at[i]:at[i + 1]], *self.held(i), window, sinks, products, bias)
            if half:
                bound = bound + HALF * want.abs() + 2.0 ** -25
            err = (got[at[i]:at[i + 1]].double() - want).abs()
            assert (err <= bound).all(), (i, float((err - bound).max()), float(err.max()), (err > bound).nonzero()[:3].tolist())


# many rows: the batch is large enough for the kernel of 256-row units (128 at head_dim 256) to be chosen
MANY = [(Q8Layout(8, 2, 128, 16, "int8"), 48, 300), (Q8Layout(32, 4, 64, 32, "e4m3"), 16, 400), (Q8Layout(14, 2, 64, 16, "int8"), 30, 300),
        (Q8Layout(12, 4, 128, 128, "e4m3"), 24, 500), (Q8Layout(6, 2, 256, 16, "int8"), 24, 300), (Q8Layout(16, 1, 256, 64, "e4m3"), 16, 300)]


@pytest.mark.parametrize("layout,batch,longest", MANY, ids=[f"{x.num_q_heads}/{x.num_kv_heads}x{x.head_dim}b{x.block_size}{x.fmt}" for x, _, _ in MANY])
def test_attention_of_prompts(layout, batch, longest, native_lib):
    rng = random.Random(batch)
    lens = [longest] + [rng.randint(1, longest) for _ in range(batch - 1)]
    lens[1], lens[2], lens[3] = 1, layout.block_size, longest - 1
    w = Large(layout, lens, 31)
    counts = [t if i % 3 else rng.randint(0, t) for i, t in enumerate(lens)]
    counts[0] = longest
    for window, sinks, half in ((0, 0, True), (0, 0, False), (33, 5, True), (longest // 2, 200, True), (1, 0, False)):
        w.check(counts, window, sinks, half, products=1)
    fewer = [min(t, 130) for t in lens]              # one tile of rows with a few in the second
    w.check(fewer, 0, 0, True, products=1)


def test_prompt_chunk_behind_a_long_cache(native_lib):
    w = Large(Q8Layout(32, 8, 128, 16, "int8"), [3000, 2100], 32)
    w.check([513, 700], window=1024, sinks=4, products=1)
    w.check([513, 700], products=1)


def test_prompts_with_masked_and_visible_poison(native_lib):
    """In the kernel for many rows: a page with a NaN scale, an infinity in a tail row of V."""
    layout, n = Q8Layout(8, 2, 128, 32, "int8"), 48
    w = Large(layout, [300] * n, 33)
    clean = w.cache
    k, v = w.k.clone(), w.v.clone()
    k[100, 1, 7] = float("nan")                      # sequence 0, page 3 (tokens 96 .. 127), kv head 1
    v[295, 0, 9] = float("inf")                      # sequence 0, tail (tokens 288 ..), kv head 0
    bad = Q8Cache(layout, clean.num_blocks, n, clean.max_blocks_per_seq, DEV)
    bad.set_block_tables(clean.block_tables)
    bad.write(k, v, i32(w.at), max_new_per_seq=300, max_start_seq_len=0)
    q = torch.randn((300 * n, 8, 128), generator=w.g, device=DEV).half()
    kw = dict(max_seq_len=300, q_offsets=i32([300 * i for i in range(n + 1)]), max_q_per_seq=300)
    outs = []
    for window in (0, 40):
        for cache in (clean, bad):
            out = torch.empty_like(q)
            cache.attend(q, out, window=window, **kw)
            outs.append(out)
    tok = torch.arange(300, device=DEV)
    for window, good, got in ((0, *outs[:2]), (40, *outs[2:])):
        assert torch.equal(got[300:], good[300:])    # the other sequences
        hit = torch.zeros((300, 8, 128), dtype=torch.bool, device=DEV)
        seen = (tok >= 96) if window == 0 else (tok >= 96) & (tok < 127 + window)
        hit[:, 4:] = seen[:, None, None]
        hit[295:, :4, 9] = True
        assert got[:300][hit].isnan().all() and torch.equal(got[:300][~hit], good[:300][~hit])


@pytest.mark.parametrize("layout,lens", [
    (Q8Layout(8, 2, 128, 16, "int8"), [20000]), (Q8Layout(10, 1, 64, 16, "e4m3"), [30000]), (Q8Layout(4, 2, 256, 32, "int8"), [9000]),
    (Q8Layout(32, 8, 128, 16, "e4m3"), [5000, 1, 4000, 300, 16, 2500]), (Q8Layout(14, 2, 64, 32, "int8"), [700] * 20 + [3, 1500]),
    (Q8Layout(32, 8, 128, 16, "int8"), [2000] * 40), (Q8Layout(16, 1, 128, 64, "int8"), [6000, 100, 3333])])
def test_contexts_cut_into_parts(layout, lens, native_lib):
    """Long contexts of few units (many parts, the merge kernel, eight-warp CTAs), of some (clusters) and of many."""
    w = Large(layout, lens, 34)
    w.check([1] * len(lens))
    w.check([1] * len(lens), half=False)
    w.check([1] * len(lens), window=1000, sinks=3)
    w.check([min(t, 3) for t in lens])


def test_a_captured_call_with_parts_and_a_captured_prompt(native_lib):
    """Two graphs, one with the merge kernel and one with the kernel for many rows, replayed in turn and on two streams."""
    w = Large(Q8Layout(10, 2, 128, 16, "int8"), [9000, 700], 36)
    many = Large(Q8Layout(8, 2, 128, 16, "int8"), [300] * 48, 37)
    q, q2 = (torch.randn((n, h, 128), generator=w.g, device=DEV).half() for n, h in ((2, 10), (300 * 48, 8)))
    mass, ends = torch.zeros((2, 2, 600), device=DEV), i32([300 * i for i in range(49)])
    calls = (lambda: w.cache.attend(q, max_seq_len=9000, page_mass=mass),
             lambda: many.cache.attend(q2, max_seq_len=300, q_offsets=ends, max_q_per_seq=300))
    eager = [c() for c in calls]
    one = mass.clone()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c())
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for k in range(6):
        for g, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, outs))
    assert ((mass - 7 * one).abs() <= 7 * 2.0 ** -22 * 7 * one + 1e-30).all()     # seven passes, six fp32 additions


def test_masses_of_a_long_context(native_lib):
    w = Large(Q8Layout(10, 2, 128, 16, "int8"), [20000, 777], 35)
    q = torch.randn((2, 10, 128), generator=w.g, device=DEV).half()
    mass = torch.zeros((2, 2, 1250), device=DEV)
    w.cache.attend(q, max_seq_len=20000, page_mass=mass)
    for i, t in enumerate(w.lens):
        k, _ = w.held(i)
        s = torch.stack([q[i, h].double() @ k[:, h // 5].T / 128 ** 0.5 for h in range(10)])
        p = torch.nn.functional.pad(torch.softmax(s, 1), (0, 20000 - t)).view(2, 5, 1250, 16).sum((1, 3))
        # a weight is off by the fp32 errors of its score, at most 2 (D + 4) 2^-24 sum|q k| / sqrt(D), here under 200, and 2^-18
        assert ((mass[i].double() - p).abs() <= (2 * 132 * 2.0 ** -24 * 200 + 2.0 ** -18) * p + 2.0 ** -40).all()
        assert abs(float(mass[i].double().sum()) - 10) < 1e-3


# ------------------------------------------------------------------------------------------------ page masses, eviction

@pytest.mark.parametrize("layout", LAYOUTS, ids=IDS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
def test_page_masses(layout, window, sinks, native_lib):
    b = layout.block_size
    lens = [1, b, b + 3, 333, 5 * b - 1]
    w = World(layout, lens, seed=16)
    w.feed(lens)
    width = max(-(-t // b) for t in lens) + 2
    start = torch.rand((len(lens), layout.num_kv_heads, width), generator=w.gen)
    mass = start.to(DEV)
    weights = w.check_attention(window=window, sinks=sinks, page_mass=mass)
    for i, (t, x) in enumerate(zip(lens, weights)):
        want = start[i].double().clone()
        want[:, :-(-t // b)] += qo.masses(x, layout.num_kv_heads, b)
        # a weight is off by the fp32 errors of its score (up to (D + 4) 2^-24 sum|q k|, here < 2^-24 * 132 * 200) and of
        # the exponential and the sums (2^-18); then one fp32 addition to the old mass
        bound = 2.0 ** -24 * want + (2 * (layout.head_dim + 4) * 2.0 ** -24 * 200 + 2.0 ** -18) * (want - start[i].double())
        assert ((mass[i].cpu().double() - want).abs() <= bound).all()
        # pages of which nothing is seen are not touched, nor columns behind the sequence
        seen = torch.zeros(width, dtype=torch.bool)
        seen[:-(-t // b)] = qo.masses(x, layout.num_kv_heads, b).sum(0) > 0
        assert torch.equal(mass[i].cpu()[:, ~seen], start[i][:, ~seen])


def random_state(gen, batch, width, nkv, block, longest):
    lens = torch.randint(0, longest + 1, (batch,), generator=gen, dtype=torch.int32)
    tables = torch.randperm(batch * width, generator=gen).to(torch.int32).view(batch, width)
    mass = torch.exp(2 * torch.randn((batch, nkv, width), generator=gen))
    mass[:, :, torch.rand(width, generator=gen) < 0.3] = 0.0      # ties
    return tables, lens, mass


@pytest.mark.parametrize("width,nkv,block,budget,first,recent", [
    (1, 1, 16, 0, 0, 0), (1, 3, 16, 1, 0, 0), (7, 2, 32, 3, 1, 1), (64, 8, 16, 30, 0, 0), (64, 8, 16, 5, 2, 3), (1000, 8, 16, 500, 1, 16),
    (1024, 1, 128, 1023, 4, 100), (1025, 2, 16, 7, 0, 7), (3000, 4, 16, 1024, 1, 16), (5000, 1, 16, 0, 0, 0), (40000, 2, 16, 12345, 3, 99)])
def test_evictions_are_exact(width, nkv, block, budget, first, recent, native_lib):
    gen = torch.Generator().manual_seed(width + budget)
    batch = 5 if width < 2000 else 3
    tables, lens, mass = random_state(gen, batch, width, nkv, block, width * block)
    lens[0], lens[1] = width * block, 0 if batch < 4 else min(width * block, budget * block + 5)
    mass[2, :, 1::3] = 1.0
    if width > 10:
        mass[0, 0, 5], mass[0, 0, 6], mass[0, 0, 7] = float("nan"), float("inf"), -0.0
    inputs = [x.to(DEV) for x in (tables, lens, mass)]
    r = evict_pages(*inputs, block_size=block, budget=budget, first=first, recent=recent, max_seq_len=width * block)
    for x, y in zip(inputs, (tables, lens, mass)):
        assert torch.equal(x.cpu().view(torch.int32), y.view(torch.int32))        # inputs stay
    for i in range(batch):
        full, left = int(lens[i]) // block, int(lens[i]) % block
        keep = qo.evict(full, mass[i], budget, first, recent)
        gone = [p for p in range(full) if p not in set(keep)]
        assert int(r.seq_lens[i]) == len(keep) * block + left
        want = torch.zeros(width, dtype=torch.int32)
        want[:len(keep)] = tables[i, keep]
        assert torch.equal(r.block_tables[i].cpu(), want)
        want = torch.full((width,), -1, dtype=torch.int32)
        want[:len(gone)] = tables[i, gone]
        assert int(r.freed_counts[i]) == len(gone) and torch.equal(r.freed[i].cpu(), want)
        columns = keep + ([full] if left else [])
        want = torch.zeros((nkv, width))
        want[:, :len(columns)] = mass[i][:, columns]
        assert torch.equal(r.page_mass[i].cpu().view(torch.int32), want.view(torch.int32))


def test_all_masses_equal_or_nan_or_infinite(native_lib):
    for value in (0.0, 1.0, float("nan"), float("inf"), float("-inf")):
        tables = torch.arange(300, dtype=torch.int32, device=DEV)[None]
        r = evict_pages(tables, i32([300 * 16 + 3]), torch.full((1, 2, 301), value, device=DEV), block_size=16, budget=100, first=2,
                        recent=8, max_seq_len=300 * 16 + 3)
        assert r.block_tables[0, :100].tolist() == list(range(92)) + list(range(292, 300))    # the lowest of equals


# ------------------------------------------------------------------------------------------------ as it is used

@pytest.mark.parametrize("layout", [LAYOUTS[0], LAYOUTS[1], LAYOUTS[2]], ids=IDS[:3])
def test_serving_run(layout, native_lib):
    """Prompts, steps with masses, an eviction, more steps over what is left: every output and the masses against the
    oracle on the rows that are still cached."""
    b, nkv = layout.block_size, layout.num_kv_heads
    lens = [9 * b + 3, 4 * b, 7 * b + b - 1]
    w = World(layout, [t + 3 * b for t in lens], seed=17)
    w.feed(lens)
    w.check_attention([min(t, 20) for t in lens], window=5 * b, sinks=2)
    mass = torch.zeros((3, nkv, w.cache.max_blocks_per_seq), device=DEV)
    want = torch.zeros(mass.shape, dtype=torch.float64)
    for _ in range(3):
        w.feed([1, 1, 1])
        for i, x in enumerate(w.check_attention(page_mass=mass)):
            part = qo.masses(x, nkv, b)
            want[i, :, :part.shape[1]] += part
    assert ((mass.cpu().double() - want).abs() <= 2.0 ** -10 * want + 1e-6).all()
    before = mass.cpu()
    r = w.cache.evict(mass, budget=5, first=1, recent=2, max_seq_len=max(w.lens()))
    held = []
    for i, (k, v) in enumerate(w.rows):
        full = k.shape[0] // b
        keep = qo.evict(full, before[i], 5, 1, 2)
        rows = [p * b + j for p in keep for j in range(b)] + list(range(full * b, k.shape[0]))
        # the cached values of what is left: pages keep their codes, the open block its rows
        k64, v64 = qo.cached(k, b, layout.fmt)[rows], qo.cached(v, b, layout.fmt)[rows]
        held.append((k64, v64))
        w.rows[i] = (k[rows], v[rows])
    assert w.cache.seq_lens.tolist() == w.lens()
    w.check_contents()
    assert sorted(r.freed[0, :int(r.freed_counts[0])].tolist()) == sorted(set(r.freed[0].tolist()) - {-1})
    w.check_attention(held=held)
    w.feed([b, 1, 2])
    w.check_contents()
    w.check_attention(window=3 * b, sinks=3, page_mass=mass)


def test_captured_steps_replay(native_lib):
    """Write + attend + masses + eviction captured once and replayed while the lengths and inputs change on the device."""
    layout = Q8Layout(8, 2, 128, 16, "int8")
    w = World(layout, [400, 400], seed=18)
    w.feed([130, 75])
    twin = World(layout, [400, 400], seed=18)
    twin.feed([130, 75], *(torch.cat([w.rows[0][j], w.rows[1][j]]) for j in (0, 1)))
    k, v, q = (torch.zeros((2, n, 128), dtype=torch.float16, device=DEV) for n in (2, 2, 8))
    out = torch.zeros((2, 8, 128), dtype=torch.float16, device=DEV)
    mass = torch.zeros((2, 2, 30), device=DEV)
    ones = i32([0, 1, 2])

    def step():
        w.cache.write(k, v, ones, max_new_per_seq=1, max_start_seq_len=399)
        w.cache.attend(q, out, max_seq_len=400, window=90, sinks=4, page_mass=mass)

    step()           # lazy set-up outside the capture; then put the state back
    w.cache.seq_lens -= 1
    mass.zero_()
    for j, (tail, mine) in enumerate(zip((w.cache.tensors.K_TAIL, w.cache.tensors.V_TAIL), (twin.cache.tensors.K_TAIL, twin.cache.tensors.V_TAIL))):
        tail.copy_(mine)
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    with torch.cuda.graph(other):
        r = evict_pages(w.cache.block_tables, w.cache.seq_lens, mass, block_size=16, budget=6, first=1, recent=2, max_seq_len=400)
    twin_mass = torch.zeros_like(mass)
    for _ in range(20):
        rows = [twin.randn(2, n, 128) for n in (2, 2, 8)]
        for dst, src in zip((k, v, q), rows):
            dst.copy_(src)
        graph.replay()
        twin.feed([1, 1], rows[0], rows[1])
        want = torch.empty_like(out)
        twin.cache.attend(rows[2].to(DEV), want, max_seq_len=400, window=90, sinks=4, page_mass=twin_mass)
        assert torch.equal(out, want) and torch.equal(mass, twin_mass)
    other.replay()
    eager = evict_pages(twin.cache.block_tables, twin.cache.seq_lens, twin_mass, block_size=16, budget=6, first=1, recent=2, max_seq_len=400)
    assert torch.equal(r.seq_lens, eager.seq_lens) and torch.equal(r.page_mass, eager.page_mass) and torch.equal(r.freed_counts, eager.freed_counts)


def test_two_streams_at_once(native_lib):
    """Two caches stepped on two streams give what each gives alone, run after run."""
    layout = Q8Layout(8, 2, 64, 16, "int8")
    worlds = [World(layout, [900, 500], seed=s) for s in (19, 20)]
    for w in worlds:
        w.feed([900, 500])
    qs = [w.randn(2, 8, 64).to(DEV) for w in worlds]
    want, base = [], []
    for w, q in zip(worlds, qs):
        m = torch.zeros((2, 2, 60), device=DEV)
        want.append(w.cache.attend(q, max_seq_len=900, page_mass=m).clone())
        base.append(m)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        got, mass = [], []
        for w, q, s in zip(worlds, qs, streams):
            with torch.cuda.stream(s):
                m = torch.zeros((2, 2, 60), device=DEV)
                got.append(w.cache.attend(q, max_seq_len=900, page_mass=m))
                mass.append(m)
        torch.cuda.synchronize()
        for a, b, c, d in zip(got, want, mass, base):
            assert torch.equal(a, b) and torch.equal(c, d)


def test_ids_and_offsets_outside_the_pools_are_refused(native_lib):
    layout = Q8Layout(4, 2, 64, 16, "int8")
    w = World(layout, [64, 64, 64], seed=21)
    w.feed([40, 40, 40])
    snapshot = [t.clone() for t in w.cache.tensors]
    torch.cuda.synchronize()
    k = w.randn(30, 2, 64).to(DEV)
    before = rejected_indices()
    tables = w.cache.block_tables.clone()

    def untouched():
        torch.cuda.synchronize()
        return all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(w.cache.tensors, snapshot))

    lens = i32([40, 40, 40])
    w.cache.block_tables[:, 2] = i32([w.cache.num_blocks, -1, 1 << 30])     # the page each would complete
    w.cache.write(k, k, i32([0, 10, 20, 30]), max_new_per_seq=10, max_start_seq_len=64, start_seq_lens=lens)
    assert untouched() and rejected_indices() == before + 3
    w.cache.block_tables.copy_(tables)
    for offsets, starts, bound in (([0, 11, 20, 30], [40, -1, 65], 10), ([-5, 5, 40, 41], [40, 40, 40], 10), ([20, 10, 31, 30], [40, 40, 40], 100)):
        w.cache.write(k, k, i32(offsets), max_new_per_seq=bound, max_start_seq_len=64, start_seq_lens=i32(starts))
    assert rejected_indices() > before + 3
    w.cache.tensors.K_TAIL.copy_(snapshot[3])
    w.cache.tensors.V_TAIL.copy_(snapshot[4])
    q = w.randn(3, 4, 64).to(DEV)
    good = w.cache.attend(q, max_seq_len=64, seq_lens=lens)
    now = rejected_indices()
    w.cache.block_tables[1, 0] = w.cache.num_blocks + 7
    got = w.cache.attend(q, max_seq_len=64, seq_lens=lens)
    assert torch.equal(got[0], good[0]) and torch.equal(got[2], good[2]) and rejected_indices() > now
    w.cache.block_tables.copy_(tables)
    got = w.cache.attend(q, max_seq_len=64, seq_lens=i32([40, -3, 40]))
    assert torch.equal(got[0], good[0]) and int(got[1].abs().max()) == 0
    good = w.cache.attend(q, max_seq_len=64, seq_lens=lens, q_offsets=i32([0, 1, 2, 3]), max_q_per_seq=8)
    out = torch.full((3, 4, 64), 5.0, device=DEV)
    w.cache.attend(q, out, max_seq_len=64, seq_lens=lens, q_offsets=i32([0, 1, 9, 3]), max_q_per_seq=8)   # rows 1..8 of 3
    assert torch.equal(out[0], good[0]) and (out[1:] == 5.0).all()
    torch.cuda.synchronize()
    now = rejected_indices()
    out.fill_(5.0)
    w.cache.attend(q, out, max_seq_len=64, seq_lens=lens, q_offsets=i32([0, 3, 3, 3]), max_q_per_seq=2)   # three rows, two stated
    assert (out == 5.0).all() and rejected_indices() == now + 1


def test_python_refusals(native_lib):
    layout = Q8Layout(4, 2, 64, 16, "int8")
    w = World(layout, [64, 64], seed=22)
    k = torch.zeros((4, 2, 64), dtype=torch.float16, device=DEV)
    offs = i32([0, 2, 4])
    kw = dict(max_new_per_seq=2, max_start_seq_len=0)
    with pytest.raises(TypeError):
        w.cache.write(k.float(), k, offs, **kw)
    with pytest.raises(RuntimeError):
        w.cache.write(k[:, :1], k, offs, **kw)
    with pytest.raises(RuntimeError):
        w.cache.write(k, k[:3], offs, **kw)
    with pytest.raises(TypeError):
        w.cache.write(k, k, offs.long(), **kw)
    with pytest.raises(RuntimeError):
        w.cache.write(k, k, offs.cpu(), **kw)
    with pytest.raises(RuntimeError):
        w.cache.write(k, k, i32([0, 1, 2, 3]), **kw)                      # more sequences than rows of the tables
    with pytest.raises(RuntimeError):
        w.cache.write(k, k, offs, slot_ids=i32([0]), **kw)
    with pytest.raises(RuntimeError):
        w.cache.write(torch.zeros((2, 64, 4), dtype=torch.float16, device=DEV).transpose(0, 2).transpose(1, 2), k, offs, **kw)
    q = torch.zeros((2, 4, 64), dtype=torch.float16, device=DEV)
    with pytest.raises(TypeError):
        w.cache.attend(q.float(), max_seq_len=64)
    with pytest.raises(TypeError):
        w.cache.attend(q, torch.empty((2, 4, 64), dtype=torch.bfloat16, device=DEV), max_seq_len=64)
    with pytest.raises(ValueError):
        w.cache.attend(q, max_seq_len=64, scale=0.0)
    with pytest.raises(RuntimeError, match="RANGE"):
        w.cache.attend(q, max_seq_len=64, window=-1)
    with pytest.raises(RuntimeError, match="BLOCK_TABLE"):
        w.cache.attend(q, max_seq_len=10000)
    mass = torch.zeros((2, 2, 4), device=DEV)
    with pytest.raises(RuntimeError):
        w.cache.attend(q, max_seq_len=64, page_mass=mass[:, :1].contiguous())
    with pytest.raises(TypeError):
        w.cache.attend(q, max_seq_len=64, page_mass=mass.double())
    with pytest.raises(RuntimeError):
        w.cache.attend(q, max_seq_len=64, page_mass=mass, q_offsets=offs[:3] // 2)
    with pytest.raises(RuntimeError, match="RANGE"):
        w.cache.evict(mass, budget=1, first=1, recent=1, max_seq_len=64)
    with pytest.raises(TypeError):
        Q8Cache.over(layout, Q8CacheTensors(*w.cache.tensors)._replace(SCALES=w.cache.tensors.SCALES.half()), w.cache.block_tables, w.cache.seq_lens)
    assert w.cache.attend(q[:0], max_seq_len=64).shape == (0, 4, 64)
    w.cache.write(k[:0], k[:0], i32([0, 0, 0]), **kw)


def test_no_bounded_wait_gave_up(native_lib):
    import ctypes
    out = ctypes.c_uint32(123)
    assert native_lib.kivi_b200_q8_wait_failures(ctypes.byref(out)) == 0 and out.value == 0
