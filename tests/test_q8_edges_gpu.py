"""The 8-bit cache's calls at their edges: masks, magnitudes, lengths and ids that the main tests do not combine."""
import pytest
import torch

from jacq_b200.q8_cache import Q8Layout, evict_pages, rejected_indices, wait_failures
from tests import q8_oracle as qo
from tests.test_q8_gpu import DEV, HALF, MANY, Large, World, i32, offsets_of

pytestmark = pytest.mark.gpu

MANY_IDS = [f"{x.num_q_heads}/{x.num_kv_heads}x{x.head_dim}b{x.block_size}{x.fmt}" for x, _, _ in MANY]


class Prompts(Large):
    """A batch large enough for the kernel for many rows, with chosen K and V instead of normal ones."""

    def fill(self, k=None, v=None):
        self.k, self.v = self.k if k is None else k.half(), self.v if v is None else v.half()
        self.cache.seq_lens.zero_()
        self.cache.write(self.k, self.v, i32(self.at), max_new_per_seq=max(self.lens), max_start_seq_len=0)
        self.scales = [float(x) for x in self.cache.tensors.SCALES.nan_to_num().amax((0, 1))]

    def positions(self):
        return torch.cat([torch.arange(t, device=DEV) for t in self.lens])

    def run(self, q, counts, half=True, **kw):
        out = torch.full(q.shape, 9.0, dtype=torch.float16 if half else torch.float32, device=DEV)
        self.cache.attend(q, out, max_seq_len=max(self.lens), q_offsets=i32(offsets_of(counts)), max_q_per_seq=max(counts), **kw)
        return out

    def compare(self, q, counts, window=0, sinks=0, half=True, products=2, some=None):
        at = offsets_of(counts)
        got = self.run(q, counts, half, window=window, sinks=sinks)
        for i in range(len(counts)) if some is None else some:
            want, bound = qo.attend_block(q[at[i]:at[i + 1]], *self.held(i), window, sinks, products)
            if half:
                bound = bound + HALF * want.abs() + 2.0 ** -25
            err = (got[at[i]:at[i + 1]].double() - want).abs()
            assert (err <= bound).all(), (i, float((err - bound).max()), float(err.max()), (err > bound).nonzero()[:3].tolist())


@pytest.mark.parametrize("layout,batch,longest", MANY, ids=MANY_IDS)
def test_prompts_whose_scores_and_v_scales_rise_all_the_time(layout, batch, longest, native_lib):
    """Every 32 keys the scores rise by 2.5 and every 16 the magnitude of V doubles (17 times, then again): the running
    maximum and V's reference are raised several times within a step and from step to step."""
    w = Prompts(layout, [longest - 3 * (i % 7) for i in range(batch)], 41)
    d, pos = layout.head_dim, w.positions()
    level = (pos // 32).float() * 2.5 / d ** 0.5
    k = level[:, None, None] + 0.05 * torch.randn(w.k.shape, generator=w.g, device=DEV)
    v = torch.randn(w.v.shape, generator=w.g, device=DEV) * torch.exp2((pos // 16 % 18).float() - 9.0)[:, None, None]
    w.fill(k, v)
    q = (1.0 + 0.05 * torch.randn((sum(w.lens), layout.num_q_heads, d), generator=w.g, device=DEV)).half()
    some = [0, 1, 5, batch - 1]
    for window, sinks, half in ((0, 0, True), (0, 0, False), (70, 3, True), (longest // 2, 40, False)):
        w.compare(q, w.lens, window, sinks, half, some=some)
    # and falling: the maximum is the first key's, V's reference the first page's
    w.fill(k.flip(0), v.flip(0))
    w.compare(q, w.lens, 0, 0, True, some=some)


@pytest.mark.parametrize("layout,batch,longest", MANY, ids=MANY_IDS)
def test_probabilities_kept_over_a_large_rise_within_a_step(layout, batch, longest, native_lib):
    """Keys 32 and 64 score 2^8 and 2^25 times the keys before them: what key 32 has left, 2^-17, is far above fp16's
    range although the factor between the two maxima, 2^-25, is not. Key 64's V is 0 in every other channel."""
    w = Prompts(layout, [longest] * batch, 43)
    pos, d = w.positions(), layout.head_dim
    level = torch.where(pos < 32, 0.5, -10.0)
    level[pos == 32], level[pos == 64] = 8.5, 25.5
    v = torch.randn(w.v.shape, generator=w.g, device=DEV)
    v[pos == 64, :, ::2] = 0.0
    w.fill((level / (d ** 0.5 * 1.4427))[:, None, None].expand_as(w.k).contiguous(), v)
    q = torch.ones((sum(w.lens), layout.num_q_heads, d), dtype=torch.float16, device=DEV)
    w.compare(q, w.lens, half=False, some=[0, batch - 1])


@pytest.mark.parametrize("layout,batch,longest", [m for m in MANY if m[0].fmt == "int8"], ids=[x for x, m in zip(MANY_IDS, MANY) if m[0].fmt == "int8"])
def test_prompts_with_a_loud_key_channel_and_pages_of_zero_keys(layout, batch, longest, native_lib):
    """A channel that q does not look at sets K's scale, so that a page's other codes are a few steps of it, and all of q
    has one sign: a score is a small sum whatever 128 sum|q| is. Every third page's K is all zero: scores exactly 0."""
    w = Prompts(layout, [longest] * batch, 42)
    k = torch.randn(w.k.shape, generator=w.g, device=DEV)
    k[..., 0] = 200.0
    page = w.positions() // layout.block_size
    k[page % 3 == 2] = 0.0
    w.fill(k)
    q = 20.0 + torch.randn((sum(w.lens), layout.num_q_heads, layout.head_dim), generator=w.g, device=DEV)
    q[..., 0] = 0.0
    some = [0, batch - 1]
    w.compare(q.half(), w.lens, some=some)
    w.compare(q.half(), w.lens, window=40, sinks=3, half=False, some=some)
    w.compare((q * 8.0).half(), w.lens, half=False, some=some)


@pytest.mark.parametrize("layout,batch,longest", MANY, ids=MANY_IDS)
def test_prompts_are_as_exact_as_single_tokens(layout, batch, longest, native_lib):
    """Probabilities to 22 bits whichever kernel runs: fp32 outputs within the bound of two fp16 numbers each."""
    w = Prompts(layout, [longest - 2 * (i % 5) for i in range(batch)], 44)
    q = torch.randn((sum(w.lens), layout.num_q_heads, layout.head_dim), generator=w.g, device=DEV).half()
    for window, sinks, half in ((0, 0, False), (0, 0, True), (90, 5, False)):
        w.compare(q, w.lens, window, sinks, half, some=[0, 3, batch - 1])


@pytest.mark.parametrize("layout,batch,longest", MANY, ids=MANY_IDS)
@pytest.mark.parametrize("power", [-14, -10, 12])
def test_prompts_with_a_tail_beside_pages_of_any_magnitude(layout, batch, longest, power, native_lib):
    """V of magnitude 2^-14 to 2^12, alike in pages and tail rows, then a tail that is 2^6 above or below its pages."""
    w = Prompts(layout, [longest - 1 - 2 * (i % 6) for i in range(batch)], 45)
    lens, b = torch.tensor(w.lens, device=DEV), layout.block_size
    v = torch.randn(w.v.shape, generator=w.g, device=DEV)
    in_tail = w.positions() >= (lens // b * b).repeat_interleave(lens)
    q = torch.randn((sum(w.lens), layout.num_q_heads, layout.head_dim), generator=w.g, device=DEV).half()
    for more in (0, 6, -6) if power < 0 else (0, -6):
        w.fill(v=v * 2.0 ** power * torch.where(in_tail, 2.0 ** more, 1.0)[:, None, None])
        w.compare(q, w.lens, 0, 0, False, some=[0, 2, batch - 1])
        w.compare(q, w.lens, 50, 3, True, some=[1])


@pytest.mark.parametrize("layout,batch,longest", MANY, ids=MANY_IDS)
def test_prompt_rows_are_not_touched_by_the_v_scales_of_keys_they_do_not_see(layout, batch, longest, native_lib):
    """V grows by 2^18 from one token on: rows before it, and rows whose window has left the large ones behind."""
    w = Prompts(layout, [longest - i % 3 for i in range(batch)], 46)
    q = torch.randn((sum(w.lens), layout.num_q_heads, layout.head_dim), generator=w.g, device=DEV).half()
    v, pos = torch.randn(w.v.shape, generator=w.g, device=DEV), w.positions()
    b = layout.block_size
    for large in (pos >= 2 * b, (pos < b) | (pos >= 3 * b), pos // b == 1):
        w.fill(v=v * torch.where(large, 2.0 ** 6, 2.0 ** -12)[:, None, None])
        w.compare(q, w.lens, 0, 0, False, some=[0, batch - 1])
        w.compare(q, w.lens, b + 5, 2, False, some=[0, 2])


@pytest.mark.parametrize("layout,batch,longest", MANY, ids=MANY_IDS)
@pytest.mark.parametrize("scale", [1e-38, 1e-33])
def test_prompts_stay_masked_under_the_smallest_scales(layout, batch, longest, scale, native_lib):
    """All scores are 0 to working precision: a row is the mean of the values that it sees, and of no other."""
    w = Prompts(layout, [longest] * batch, 47)
    q = torch.randn((sum(w.lens), layout.num_q_heads, layout.head_dim), generator=w.g, device=DEV).half()
    got = w.run(q, w.lens, half=False, scale=scale)[:longest].double()
    v, per = w.held(0)[1], layout.num_q_heads // layout.num_kv_heads
    count = torch.arange(1, longest + 1, device=DEV)[:, None, None]
    want = (v.cumsum(0) / count).repeat_interleave(per, 1)
    # 2^-22 of each probability and 2^-18 for the sums, as in the oracle's bound
    bound = 2.0 ** -17 * (v.abs().cumsum(0) / count).repeat_interleave(per, 1) + longest * 2.0 ** -30 * v.abs().max()
    assert ((got - want).abs() <= bound).all()


# ------------------------------------------------------------------------------------------------ evictions

def test_an_installed_eviction_keeps_the_pages_entered_for_growth(native_lib):
    """Ids behind a sequence's complete pages stay its own: every id is kept, freed or still assigned, new blocks go to
    the ids entered for them, and page 0, which another sequence holds, is not written."""
    layout, b = Q8Layout(4, 2, 64, 16, "int8"), 16
    w = World(layout, [12 * b, 12 * b, 12 * b], seed=60, spare=0)
    tables = torch.randperm(36, generator=w.gen).to(torch.int32).view(3, 12)
    zero = (tables == 0).nonzero()[0]
    tables[zero[0], zero[1]], tables[1, 2] = tables[1, 2].clone(), 0      # page 0: the third page of sequence 1
    w.cache.set_block_tables(tables)
    w.feed([7 * b + 5, 9 * b, 3 * b + 1])
    mass = torch.rand((3, 2, 12), generator=w.gen)
    mass[1, :, 2] = 9.0                                                   # kept
    r = w.cache.evict(mass.to(DEV), budget=4, first=1, recent=1, max_seq_len=9 * b)
    after = w.cache.block_tables.cpu()
    for i, full in enumerate((7, 9, 3)):
        kept = min(4, full)
        freed = r.freed[i, :int(r.freed_counts[i])].tolist()
        assert torch.equal(after[i, :kept], r.block_tables[i, :kept].cpu()) and int(r.block_tables[i, kept:].abs().max()) == 0
        assert after[i, kept:12 - full + kept].tolist() == tables[i, full:].tolist()
        assert (after[i, 12 - full + kept:] == -1).all()
        assert sorted(after[i, :12 - full + kept].tolist() + freed) == sorted(tables[i].tolist())
    assert 0 in after[1, :4]
    codes, scales = (x.clone() for x in (w.cache.tensors.K_PAGES.view(torch.int8)[0], w.cache.tensors.SCALES[0]))
    keep = [qo.evict(n // b, mass[i], 4, 1, 1) for i, n in enumerate(w.lens())]
    for i, (k, v) in enumerate(w.rows):
        rows = [p * b + j for p in keep[i] for j in range(b)] + list(range(k.shape[0] // b * b, k.shape[0]))
        w.rows[i] = (k[rows], v[rows])
    w.check_contents()
    w.feed([2 * b, 2 * b + 3, b - 1])                                     # complete blocks in the pages entered before
    w.check_contents()
    assert torch.equal(codes, w.cache.tensors.K_PAGES.view(torch.int8)[0]) and torch.equal(scales, w.cache.tensors.SCALES[0])
    # past the pages that were entered: refused and counted, and no page is written
    before, pages = rejected_indices(), [t.clone() for t in w.cache.tensors[:3]]
    rows = w.randn(8 * b, 2, 64).to(DEV)
    w.cache.write(rows, rows, i32([0, 0, 8 * b, 8 * b]), max_new_per_seq=8 * b, max_start_seq_len=12 * b, start_seq_lens=w.cache.seq_lens)
    assert rejected_indices() == before + 1
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(pages, w.cache.tensors))


def test_an_installed_eviction_that_evicts_nothing_changes_no_table(native_lib):
    layout = Q8Layout(4, 2, 64, 16, "e4m3")
    w = World(layout, [100, 60], seed=61)
    w.feed([50, 60])
    tables = w.cache.block_tables.clone()
    w.cache.evict(torch.ones((2, 2, w.cache.max_blocks_per_seq), device=DEV), budget=50, max_seq_len=100)
    assert torch.equal(tables, w.cache.block_tables) and w.cache.seq_lens.tolist() == [50, 60]


def test_evictions_let_lengths_outside_the_bounds_through(native_lib):
    """A sequence longer than max_seq_len, or of negative length: nothing is cut, freed or moved, and it is counted."""
    width, gen = 20, torch.Generator().manual_seed(62)
    lens = [160, 161, 20 * 16, -1, 0, 20 * 16 + 5]
    tables = torch.randperm(6 * width, generator=gen).to(torch.int32).view(6, width)
    mass = torch.rand((6, 2, width), generator=gen)
    before = rejected_indices()
    r = evict_pages(tables.to(DEV), i32(lens), mass.to(DEV), block_size=16, budget=4, first=1, recent=1, max_seq_len=160)
    assert rejected_indices() == before + 4
    assert r.seq_lens.tolist() == [64, 161, 320, -1, 0, 325]
    assert r.freed_counts.tolist() == [6, 0, 0, 0, 0, 0]
    for i in (1, 2, 3, 5):
        assert torch.equal(r.block_tables[i].cpu(), tables[i]) and torch.equal(r.page_mass[i].cpu(), mass[i])
        assert (r.freed[i] == -1).all()
    # and so does an installed one
    layout = Q8Layout(4, 2, 64, 16, "int8")
    w = World(layout, [200, 90], seed=63)
    w.feed([200, 90])
    tables, mass = w.cache.block_tables.clone(), torch.rand((2, 2, w.cache.max_blocks_per_seq), device=DEV)
    kept = mass.clone()
    r = w.cache.evict(mass, budget=3, max_seq_len=100)
    assert torch.equal(w.cache.block_tables[0], tables[0]) and w.cache.seq_lens.tolist() == [200, 58] and torch.equal(mass[0], kept[0])
    assert int(r.freed_counts[1]) == 2


# ------------------------------------------------------------------------------------------------ writer

@pytest.mark.parametrize("layout", [Q8Layout(8, 2, 128, 16, "int8"), Q8Layout(3, 3, 64, 32, "e4m3"), Q8Layout(4, 2, 256, 128, "int8")], ids=["16", "32", "128"])
def test_the_writer_leaves_tail_rows_behind_the_last_token(layout, native_lib):
    """A call writes the rows of its own tokens that stay open and no other row of the slot, nor another slot's."""
    b = layout.block_size
    w = World(layout, [4 * b] * 5, seed=72)
    mark = 0x7abc                                  # a NaN that no arithmetic leaves
    tails = (w.cache.tensors.K_TAIL, w.cache.tensors.V_TAIL)
    for tail in tails:
        tail.view(torch.int16).fill_(mark)
    written = [0] * 5                              # rows of the slot that have ever been written
    for counts in ([0, 1, b - 1, b, b + 3], [0, b - 2, 0, 1, 2 * b - 6], [0, 2, 2, 0, 1]):
        before = w.lens()
        w.feed(counts)
        for i, (old, n) in enumerate(zip(before, counts)):
            end = (old + n) % b
            if n:
                written[i] = max(written[i], end) if (old + n) // b > old // b else max(written[i], old % b + n)
            for tail in tails:
                rows = tail[i].view(torch.int16).cpu()
                assert (rows[:, written[i]:] == mark).all() and (end == 0 or not (rows[:, :end] == mark).all(-1).any())
    w.check_contents()


# ------------------------------------------------------------------------------------------------ lengths, ids, bounds

@pytest.mark.parametrize("many", [False, True])
def test_attention_counts_lengths_outside_the_bounds(many, native_lib):
    """In both kernels a length above max_seq_len answers as max_seq_len, a negative one as 0, and each is counted once."""
    layout, batch, longest = MANY[0]
    w = Prompts(layout, [longest] * batch, 64)
    lens = [longest] * batch
    lens[1], lens[4], lens[7] = longest + 1, -5, 1 << 29
    clamped = [min(max(t, 0), longest) for t in lens]
    n = longest if many else 1
    q = torch.randn((n * batch, layout.num_q_heads, layout.head_dim), generator=w.g, device=DEV).half()
    kw = dict(max_seq_len=longest, q_offsets=i32([n * i for i in range(batch + 1)]), max_q_per_seq=n) if many else dict(max_seq_len=longest)
    before = rejected_indices()
    good = w.cache.attend(q, seq_lens=i32(clamped), **kw)
    assert rejected_indices() == before
    assert torch.equal(w.cache.attend(q, seq_lens=i32(lens), **kw), good) and rejected_indices() == before + 3
    assert int(good[4 * n:5 * n].abs().max()) == 0
    if not many:
        mass = torch.zeros((batch, layout.num_kv_heads, w.cache.max_blocks_per_seq), device=DEV)
        w.cache.attend(q, seq_lens=i32(lens), page_mass=mass, **kw)
        assert rejected_indices() == before + 6


@pytest.mark.parametrize("window", [(1 << 31) - 2, (1 << 31) - 1, 1 << 30])
def test_the_largest_windows_hide_nothing_from_runs_longer_than_their_sequence(window, native_lib):
    w = World(Q8Layout(4, 2, 128, 16, "int8"), [40], seed=65)
    w.feed([40])
    q = w.randn(60, 4, 128)                       # tokens -20 .. 39
    want = w.attend(q, [60])
    assert torch.equal(w.attend(q, [60], window=window), want) and torch.equal(w.attend(q, [60], window=window, sinks=(1 << 31) - 1), want)


@pytest.mark.parametrize("layout", [Q8Layout(8, 2, 128, 32, "int8"), Q8Layout(6, 1, 64, 64, "e4m3"), Q8Layout(12, 1, 256, 16, "int8")],
                         ids=["128", "64", "256"])
def test_a_nan_in_a_visible_tail_row_shows_whatever_its_weight(layout, native_lib):
    """Its key scores e^-60 below the others: the weight underflows, a NaN times it does not."""
    b, d = layout.block_size, layout.head_dim
    t = 2 * b + 10
    w = World(layout, [t], seed=66)
    k, v = w.randn(t, layout.num_kv_heads, d), w.randn(t, layout.num_kv_heads, d)
    k[t - 4] = -60.0 / d ** 0.5
    v[t - 4, 0, 5] = float("nan")
    v[t - 4, 0, 6] = float("-inf")
    w.feed([t], k, v)
    per = layout.num_q_heads // layout.num_kv_heads
    for n, window in ((1, 0), (1, 4), (1, 3), (7, 0), (7, 3)):
        got = w.attend(torch.ones((n, layout.num_q_heads, d)).half(), None if n == 1 else [n], window=window)
        bad = torch.zeros(got.shape, dtype=torch.bool)
        for i, at in enumerate(range(t - n, t)):                        # token t - 4 is seen from itself on, as long as the window
            if at >= t - 4 and (window == 0 or t - 4 > at - window):
                bad[i, :per, 5:7] = True
        assert torch.equal(got.isnan(), bad), (n, window)


def test_slots_that_are_not_there_are_refused_by_every_call(native_lib):
    """Slot ids outside the tables: nothing is written or advanced, rows stay, attention gives zeros; each is counted."""
    layout = Q8Layout(4, 2, 64, 16, "int8")
    w = World(layout, [90, 90, 90], seed=67)
    w.feed([40, 50, 64])
    ids = i32([2, -1, 0, 3, 1 << 30])
    k, q = w.randn(5, 2, 64).to(DEV), w.randn(5, 4, 64).to(DEV)
    before = rejected_indices()
    good = w.cache.attend(q[[0, 2]], max_seq_len=90, slot_ids=i32([2, 0]))
    got = w.cache.attend(q, max_seq_len=90, slot_ids=ids)
    assert torch.equal(got[[0, 2]], good) and int(got[[1, 3, 4]].abs().max()) == 0 and rejected_indices() == before + 3
    got = w.cache.attend(q, max_seq_len=90, slot_ids=ids, seq_lens=i32([64, 40, 40, 40, 40]))     # the caller's lengths
    assert torch.equal(got[[0, 2]], good) and int(got[[1, 3, 4]].abs().max()) == 0 and rejected_indices() == before + 6
    out = [torch.full((5, 2, 64), 3.0, dtype=torch.float16, device=DEV) for _ in range(2)]
    w.cache.read(i32([0, 1, 2, 3, 4, 5]), i32([5] * 5), total=5, max_rows_per_seq=1, slot_ids=ids, k_out=out[0], v_out=out[1])
    assert (out[0][[1, 3, 4]] == 3.0).all() and not (out[0][[0, 2]] == 3.0).any() and rejected_indices() == before + 9
    w.cache.write(k, k, i32([0, 1, 2, 3, 4, 5]), max_new_per_seq=1, max_start_seq_len=90, slot_ids=ids)
    assert w.cache.seq_lens.tolist() == [41, 50, 65] and rejected_indices() == before + 12
    w.rows = [(torch.cat([a, b]), torch.cat([c, b])) for (a, c), b in zip(w.rows, (k[2:3].cpu(), k[:0].cpu(), k[:1].cpu()))]
    w.check_contents()
    graph, lens, ends = torch.cuda.CUDAGraph(), w.cache.seq_lens.clone(), i32([0, 1, 2, 3, 4, 5])
    with torch.cuda.graph(graph):
        w.cache.write(k, k, ends, max_new_per_seq=1, max_start_seq_len=90, slot_ids=ids)
        got = w.cache.attend(q, max_seq_len=90, slot_ids=ids)
    graph.replay()
    assert (w.cache.seq_lens - lens).tolist() == [1, 0, 1]
    assert torch.equal(got[[0, 2]], w.cache.attend(q[[0, 2]], max_seq_len=90, slot_ids=i32([2, 0])))


def test_a_growing_context_leaves_no_growing_state(native_lib):
    w = World(Q8Layout(8, 2, 64, 16, "int8"), [900], seed=68)
    w.feed([900])
    q = w.randn(1, 8, 64).to(DEV)
    mass = torch.zeros((1, 2, w.cache.max_blocks_per_seq), device=DEV)
    lens, seen = i32([300]), set()
    want = w.cache.attend(q, max_seq_len=300, seq_lens=lens)
    for t in range(300, 800):
        got = w.cache.attend(q, max_seq_len=t, seq_lens=lens, page_mass=mass)
        # other parts, other orders of fp32 sums of 300 weights and values below 8: 2^-18 each, and masses do not enter
        assert t % 100 or float((got - want).abs().max()) <= 8 * 2.0 ** -17
        seen.add(len(w.cache._workspace_bytes))
    assert max(seen) <= 64


def test_rows_that_nobody_writes_are_zeros_in_an_output_of_the_calls_own(native_lib):
    """Rows behind the last sequence, before the first, and of a sequence that is refused."""
    w = World(Q8Layout(4, 2, 64, 16, "int8"), [30, 30, 30], seed=69)
    w.feed([30, 30, 30])
    q = w.randn(12, 4, 64).to(DEV)
    ends = i32([2, 4, 10, 11])                   # rows 0, 1 and 11 belong to nobody; the second sequence has six, four are stated
    given = torch.full(q.shape, 5.0, device=DEV)
    w.cache.attend(q, given, max_seq_len=30, q_offsets=ends, max_q_per_seq=4)
    for _ in range(4):                           # the allocator's old blocks hold something
        torch.full(q.shape, float("nan"), device=DEV)
        got = w.cache.attend(q, max_seq_len=30, q_offsets=ends, max_q_per_seq=4)
        nobody = (given == 5.0).all(-1).all(-1)
        assert nobody.tolist() == [True] * 2 + [False] * 2 + [True] * 6 + [False, True]
        assert int(got[nobody].abs().max()) == 0 and torch.equal(got[~nobody], given[~nobody])


def test_no_wait_gave_up(native_lib):
    assert wait_failures() == 0


def test_an_eviction_wants_the_caches_own_masses(native_lib):
    w = World(Q8Layout(4, 2, 64, 16, "int8"), [64, 64], seed=70)
    w.feed([64, 64])
    tables = w.cache.block_tables.clone()
    for shape in ((2, 1, 4), (2, 3, 4), (1, 2, 4)):
        with pytest.raises(RuntimeError, match="page_mass"):
            w.cache.evict(torch.zeros(shape, device=DEV), budget=1, max_seq_len=64)
    assert torch.equal(tables, w.cache.block_tables) and w.cache.seq_lens.tolist() == [64, 64]


@pytest.mark.parametrize("heads", [1, 3, 5, 11])
def test_an_infinite_key_of_no_weight_leaves_the_masses_finite(heads, native_lib):
    """K's tail holds -infinity where q is positive: weight 0. Query rows a unit has room for and nobody fills are 0, and
    0 times infinity is no number."""
    layout = Q8Layout(2 * heads, 2, 64, 32, "int8")
    w = World(layout, [48], seed=71)
    k, v = w.randn(48, 2, 64), w.randn(48, 2, 64)
    k[40, :, 3] = float("-inf")
    w.feed([48], k, v)
    q = w.randn(1, 2 * heads, 64)
    q[..., 3] = q[..., 3].abs() + 0.1
    mass = torch.zeros((1, 2, 2), device=DEV)
    out = w.attend(q, page_mass=mass)
    held = w.held()[0]
    keep = [t for t in range(48) if t != 40]
    s = torch.einsum("hd,thd->ht", q[0].double(), held[0].repeat_interleave(heads, 1)[keep]) / 8.0
    p = torch.zeros((2 * heads, 48), dtype=torch.float64)
    p[:, keep] = torch.softmax(s, 1)
    want = torch.nn.functional.pad(p, (0, 16)).view(2, heads, 2, 32).sum((1, 3))
    assert out.isfinite().all() and ((mass[0].cpu().double() - want).abs() <= 2.0 ** -14 * want + 1e-12).all()
