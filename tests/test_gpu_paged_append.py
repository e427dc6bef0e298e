"""GPU: rows that enter the paged cache (b200fc_kv_append) against the formula in 64 bits, and append and attention together."""
import pytest
import torch

from mm_amx_b200 import capi
from paged_cases import BF16, Paged

pytestmark = pytest.mark.gpu


def tables(positions, rot, gap=0):
    t = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) / max(1, rot // 2))
    wide = torch.full((2, positions, rot // 2 + gap), float("nan"), device="cuda")
    wide[0, :, :rot // 2], wide[1, :, :rot // 2] = t.cos(), t.sin()
    return wide


def append(c, rot=0, interleaved=False, axes=1, section=(0, 0, 0), positions=None, turns=None, with_q=True, in_place=False, stream=None, **kw):
    """the rows of c.wide: its first heads are q, then k, then v"""
    k, v = c.wide[:, c.H:c.H + c.Hkv], c.wide[:, c.H + c.Hkv:]
    cache = c.cache()
    rs, hs = c.wide.stride(0) * 2, c.wide.stride(1) * 2
    a = dict(cache=capi.pointer(cache), T=c.T, row_start=None if c.row_start is None else c.row_start.data_ptr(), k=k.data_ptr(), k_row_stride=rs, k_head_stride=hs,
             v=v.data_ptr(), v_row_stride=rs, v_head_stride=hs, rot_dim=rot, interleaved=int(interleaved), axes=axes, section=(capi.c_int * 3)(*section))
    if with_q:
        o = c.q if in_place else c.out
        a.update(H=c.H, q=c.q.data_ptr(), q_row_stride=rs, q_head_stride=hs, q_out=o.data_ptr(), q_out_row_stride=o.stride(0) * 2, q_out_head_stride=o.stride(1) * 2)
    if rot:
        a.update(rot_positions=turns.shape[1], rot_cos=turns[0].data_ptr(), rot_sin=turns[1].data_ptr(), rot_stride=turns.stride(1) * 4)
    if positions is not None:
        a.update(positions=positions.data_ptr(), position_stride=positions.stride(0) * 4)
    a.update(kw)
    capi.kv_append(capi.KvAppend(**a), stream=stream)


def turned(x, at, rot, interleaved, turns):
    """x [T, heads, D] turned by the angles at[T, rot / 2] of the tables, and |a| + |b| of each component's pair"""
    x = x.double()
    y, mag = x.clone(), x.abs()
    if rot:
        pair = torch.arange(rot // 2, device="cuda")
        cos, sin = (turns[i].double()[at, pair][:, None] for i in range(2))
        i, j = (2 * pair, 2 * pair + 1) if interleaved else (pair, pair + rot // 2)
        a, b = x[..., i], x[..., j]
        y[..., i], y[..., j] = a * cos - b * sin, b * cos + a * sin
        mag[..., i] = mag[..., j] = a.abs() + b.abs()
    return y, mag


def angles(c, rot, axes, section, positions):
    place = torch.zeros(c.T, dtype=torch.long, device="cuda")
    for b in range(c.B):
        place[c.starts[b]:c.starts[b + 1]] = torch.arange(c.lens[b] - c.rows[b], c.lens[b], device="cuda")
    if positions is None:
        return place, place.clamp(min=0)[:, None].expand(-1, rot // 2)
    axis = [0] * (rot // 2) if axes == 1 else [a for a in range(3) for _ in range(section[a])]
    return place, positions.long()[torch.tensor(axis, dtype=torch.long, device="cuda")].T if rot else positions.long()[:1].T[:, :0]


def check_append(c, rot=0, interleaved=False, axes=1, section=(0, 0, 0), positions=None, turns=None, with_q=True, in_place=False):
    """runs the call and compares q, every byte of the pool and every factor"""
    before = [t.clone() for t in c.raw]
    factors = [t.clone() for t in c.scales] if c.int8 else None
    place, at = angles(c, rot, axes, section, positions)
    q, qm = turned(c.q, at, rot, interleaved, turns)
    k, km = turned(c.wide[:, c.H:c.H + c.Hkv], at, rot, interleaved, turns)
    v = c.wide[:, c.H + c.Hkv:].double()
    append(c, rot, interleaved, axes, section, positions, turns, with_q, in_place)
    capi.sync_check()
    owned = torch.zeros(c.T, dtype=torch.bool, device="cuda")
    owned[c.starts[0]:c.starts[-1]] = True
    owned &= place >= 0
    if with_q:
        got = (c.q if in_place else c.out[:, :c.H]).double()
        # the products and their sum are rounded to fp32, then the sum once to bf16
        assert bool(((got - q).abs() <= BF16 * q.abs() * (1 + 2 ** -7) + 2 ** -22 * qm)[owned].all())
        if not in_place:
            assert bool((got[~owned] == 7.0).all()) and bool((c.out[:, c.H:] == 7.0).all())
    same = [torch.ones(t.shape, dtype=torch.bool, device="cuda") for t in c.raw]       # what must not change
    for i, (new, mag) in enumerate(((k, km), (v, v.abs()))):
        pool, was = c.pool[i], before[i].as_strided(c.pool[i].shape, c.pool[i].stride())
        keep = same[i].as_strided(c.pool[i].shape, c.pool[i].stride())
        for b in range(c.B):
            for j, pg in enumerate(c.ids[b]):
                lo, hi = max(0, c.lens[b] - c.rows[b], j * c.P), min(c.lens[b], (j + 1) * c.P)
                if lo >= hi:
                    continue
                r = slice(c.starts[b] + lo - (c.lens[b] - c.rows[b]), c.starts[b] + hi - (c.lens[b] - c.rows[b]))
                want, m = new[r].transpose(0, 1), mag[r].transpose(0, 1)
                got = pool[pg, :, lo - j * c.P:hi - j * c.P].double()
                keep[pg, :, lo - j * c.P:hi - j * c.P] = False
                if not c.int8:
                    assert bool(((got - want).abs() <= BF16 * want.abs() * (1 + 2 ** -7) + 2 ** -22 * m).all())
                    continue
                old = lo - j * c.P
                s0 = factors[i][pg, :c.Hkv].double() if old else torch.zeros(c.Hkv, dtype=torch.float64, device="cuda")
                s = torch.maximum(s0, want.abs().amax((1, 2)) / 127)
                s = torch.where(s < 2.0 ** -126, 0, s)               # (by definition: their reciprocal is no number of fp32)
                f = c.scales[i][pg, :c.Hkv].double()
                assert bool(((f - s).abs() <= 2 ** -21 * (s + m.amax((1, 2)) / 127)).all())
                # half a step of the stored integers; 127 * 2^-21 for the fp32 products and the reciprocal, and what the rotation's fp32 does
                # to a value in steps.  A factor below fp32's normal numbers is 0, and so are the integers
                none = (f == 0)[:, None, None]
                assert bool((want.abs() < 128 * 2.0 ** -126)[none.expand_as(want)].all())
                step = torch.where(none, 1, f[:, None, None])
                slack = 0.5 + 127 * 2 ** -21 + 2 ** -22 * (m / step)
                assert bool(((got - torch.where(none, 0, want) / step).abs() <= slack).all())
                if old:
                    grown = f > s0
                    was_old, now = was[pg, :, :old].double(), pool[pg, :, :old].double()
                    assert torch.equal(now[~grown], was_old[~grown])
                    assert bool(((now - was_old.clamp(min=-127) * (s0 / f)[:, None, None]).abs() <= 0.5 + 127 * 2 ** -21 + 1e-30)[grown & (s0 == s0)].all())
                    keep[pg, :, :old] &= ~grown[:, None, None]
        assert torch.equal(c.raw[i][same[i]].view(torch.int8), before[i][same[i]].view(torch.int8))
        if c.int8:
            assert bool(torch.isnan(c.scales[i][:, c.Hkv:]).all())
    return k, v


ROWS = [([1, 1, 1, 1, 1], [1, 16, 17, 40, 0]), ([1] * 40, [7 * i + 1 for i in range(40)]), ([5, 0, 33, 1], [5, 9, 70, 128]), ([100, 300], [90, 517]), ([64, 16, 200], [64, 32, 200])]


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("rows,lens", ROWS, ids=["one", "many", "few", "front", "aligned"])
@pytest.mark.parametrize("Hkv,G,D,page,rot,interleaved", [(2, 4, 128, 16, 128, False), (1, 3, 64, 64, 64, True), (3, 1, 128, 128, 32, False), (2, 2, 64, 32, 48, True), (8, 4, 128, 32, 0, False)])
def test_append(rows, lens, Hkv, G, D, page, rot, interleaved, int8):
    one = all(r == 1 for r in rows)
    c = Paged(rows, lens, Hkv, G, D, page, int8, extra=0 if one else 3, row0=0 if one else 2, one_row=one)
    check_append(c, rot, interleaved, turns=tables(max(lens) + 1, rot, 4))


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("axes,section", [(1, (0, 0, 0)), (3, (16, 24, 24)), (3, (11, 0, 53)), (3, (0, 64, 0))])
def test_given_positions(axes, section, interleaved, int8):
    c = Paged([20, 7], [50, 7], 2, 2, 128, 16, int8)
    positions = torch.randint(0, 5000, (axes, c.T), generator=c.g, device="cuda", dtype=torch.int32)
    check_append(c, 128, interleaved, axes, section, positions, tables(5000, 128))


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_q_in_place_and_without_q(int8):
    for rot, interleaved in ((128, False), (64, True)):
        c = Paged([20, 1], [33, 90], 2, 4, 128, 32, int8)
        check_append(c, rot, interleaved, turns=tables(100, rot), in_place=True)
        c = Paged([20, 1], [33, 90], 2, 4, 128, 32, int8)
        check_append(c, rot, interleaved, turns=tables(100, rot), with_q=False)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("layout", ["places", "padded"])
def test_layouts(layout, int8):
    c = Paged([20, 1, 50], [33, 90, 50], 3, 2, 64, 16, int8, layout=layout)
    check_append(c, 64, False, turns=tables(100, 64, 8))


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_sequences_that_share_pages_none_writes(int8):
    """what several sequences begin with stays as it is"""
    c = Paged([20, 1, 33], [90, 81, 97], 2, 2, 64, 16, int8)
    for b in (1, 2):
        c.ids[b][:4] = c.ids[0][:4]
        c.table[b, :4] = c.table[0, :4]
    check_append(c)


def test_factors_that_grow_and_stay():
    """new values smaller than a page's, larger, all zero, and values whose factor is too small for fp32"""
    for std in (0.0, 1e-3, 1.0, 50.0, 1e-39):
        c = Paged([1, 1, 3, 20], [5, 17, 40, 45], 2, 2, 64, 16, True)
        c.wide.mul_(std)
        check_append(c)
        if std in (0.0, 1e-39):
            assert float(c.scales[0][c.ids[2][1:], :2].abs().max()) > 0.0 and float(c.scales[0][c.ids[3][2:], :2].abs().max()) == 0.0


def test_infinities_and_nan_mark_their_page():
    for what in (float("inf"), float("-inf"), float("nan")):
        c = Paged([4, 20], [30, 20], 2, 2, 64, 16, True)
        c.wide[2, c.H + 1, 7] = what             # k of head 1, token 28 of sequence 0
        c.wide[4 + 17, c.H + 2 + 0, 3] = what    # v of head 0, token 17 of sequence 1
        append(c)
        capi.sync_check()
        ks, vs = c.scales[0][:, :2], c.scales[1][:, :2]
        assert torch.isnan(ks[c.ids[0]]).tolist() == [[False, False], [False, True]]
        assert torch.isnan(vs[c.ids[1]]).tolist() == [[False, False], [True, False]]
        assert not torch.isnan(ks[c.ids[1]]).any() and not torch.isnan(vs[c.ids[0]]).any()
        # ... and stay there until the page starts anew
        c.wide.fill_(0.5)
        append(c)
        capi.sync_check()
        assert torch.isnan(c.scales[0][c.ids[0][1], 1]) and not torch.isnan(c.scales[1][c.ids[1], :2]).any()


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_what_is_out_of_range_is_reported_and_left_out(int8):
    c = Paged([20, 3, 1], [40, 60, 17], 2, 2, 64, 16, int8)
    turns = tables(100, 64)
    keep_rows, keep_lens, keep_table = c.row_start.clone(), c.seq_lens.clone(), c.table.clone()

    def broken(unharmed):
        pools, factors = [t.clone() for t in c.raw], [t.clone() for t in c.scales or []]
        append(c, 64, turns=turns)
        with pytest.raises(capi.B200FCError) as e:
            capi.sync_check()
        assert e.value.code == capi.ERR_INVALID
        for i in range(2):
            was = pools[i].as_strided(c.pool[i].shape, c.pool[i].stride())
            assert torch.equal(c.pool[i][unharmed].view(torch.int8), was[unharmed].view(torch.int8))
        c.row_start.copy_(keep_rows); c.seq_lens.copy_(keep_lens); c.table.copy_(keep_table)

    spare = [p for p in range(c.pages) if not any(p in ids for ids in c.ids)]
    for entry in (-1, c.pages, 2 ** 31 - 1):
        c.table[1, 3] = entry
        broken(spare + c.ids[1])
    for n in (-1, 2 ** 31 - 1, c.table.shape[1] * 16 + 1):
        c.seq_lens[0] = n
        broken(spare + c.ids[0])
    for last in (c.T + 1, -1, -2 ** 31):
        c.row_start[3] = last
        broken(spare + c.ids[2])
    positions = torch.full((1, c.T), 99, dtype=torch.int32, device="cuda")
    for at in (100, -1, 2 ** 31 - 1):
        positions[0, 5] = at
        append(c, 64, positions=positions, turns=turns)
        with pytest.raises(capi.B200FCError):
            capi.sync_check()
        assert torch.equal(c.out[5, :c.H], c.q[5])                # turned by nothing
    capi.sync_check()


@pytest.mark.parametrize("with_q", [True, False])
@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("rows", [[0 if b % 5 == 2 else 3 for b in range(300)], [1] * 32 + [0] * 40, [0, 0, 2]], ids=["many", "none behind", "few"])
def test_every_sequence_outside_its_buffers_is_reported(rows, int8, with_q):
    """wherever it stands among the call's sequences, with rows or without; the others' pages are filled as without it"""
    n = len(rows)
    c, want = (Paged(rows, [9 + b % 7 for b in range(n)], 1, 2, 64, 16, int8) for _ in range(2))
    append(want, with_q=with_q)
    capi.sync_check()
    starts, lens = c.row_start.clone(), c.seq_lens.clone()

    def broken(harmed):
        append(c, with_q=with_q)
        with pytest.raises(capi.B200FCError) as e:
            capi.sync_check()
        assert e.value.code == capi.ERR_INVALID
        c.row_start.copy_(starts); c.seq_lens.copy_(lens)
        fine = [pg for b in range(n) if b not in harmed for pg in c.ids[b]]
        for i in range(2):
            assert torch.equal(c.pool[i][fine].view(torch.int8), want.pool[i][fine].view(torch.int8))

    for b in sorted({0, 2 % n, 33 % n, 137 % n, n - 3, n - 1}):
        for length in (-1, 2 ** 31 - 1, c.table.shape[1] * 16 + 1):
            c.seq_lens[b] = length
            broken([b])
    c.row_start[n] = c.T + 1
    broken([n - 1])
    c.row_start[n - 1] = -1
    broken(range(n))                     # (where row_start falls, rows of other sequences may not be found)
    c.row_start[n - 1] = c.T + 1
    broken([n - 2, n - 1])


def test_captured_and_replayed():
    """lengths and pages move on between replays"""
    for int8 in (False, True):
        c = Paged([1, 1], [16, 30], 2, 2, 64, 16, int8, one_row=True)
        turns = tables(100, 64)
        s = torch.cuda.Stream()
        append(c, 64, turns=turns, stream=s.cuda_stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            append(c, 64, turns=turns, stream=s.cuda_stream)
        other = Paged([1, 1], [16, 30], 2, 2, 64, 16, int8, one_row=True)
        spare = [p for p in range(c.pages) if not any(p in ids for ids in c.ids)]
        for x in (c, other):
            x.lens = [17, 31]
            x.seq_lens += 1
            x.ids[0] = x.ids[0] + spare[:1]
            x.table[0, 1] = spare[0]
        # (c has had its first tokens once more; the other cache gets them now)
        other.lens, other.seq_lens[:] = [16, 30], torch.tensor([16, 30], dtype=torch.int32, device="cuda")
        append(other, 64, turns=turns)
        other.lens, other.seq_lens[:] = [17, 31], torch.tensor([17, 31], dtype=torch.int32, device="cuda")
        append(other, 64, turns=turns)
        graph.replay()
        torch.cuda.synchronize()
        capi.sync_check()
        for b in range(2):
            for i in range(2):
                assert torch.equal(c.cached(i, b), other.cached(i, b))


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_a_prompt_in_chunks_then_tokens_one_by_one(int8, window, sinks):
    """append and attention together, as a program serves: two sequences, chunks of their prompts, then single tokens.  Against attention over what the
    cache holds (in 64 bits) each time, and what it holds against the rotated rows"""
    Hkv, G, D, P = 2, 4, 128, 16
    steps = [[70, 33], [130, 0], [1, 20], [1, 1], [1, 1], [1, 1], [3, 5], [1, 1]]
    total = [sum(s[b] for s in steps) for b in range(2)]
    whole = Paged(total, total, Hkv, G, D, P, int8)                # pages and tables for everything
    for i in range(2):
        whole.raw[i].fill_(77 if int8 else float("nan"))
    turns = tables(max(total), D)
    x = [whole.wide[whole.starts[b]:whole.starts[b] + total[b]].clone() for b in range(2)]
    done = [0, 0]
    for step in steps:
        c = whole
        c.rows, c.lens = step, [done[b] + step[b] for b in range(2)]
        c.starts = [0, step[0], step[0] + step[1]]
        c.T = c.starts[-1]
        c.row_start.copy_(torch.tensor(c.starts))
        c.seq_lens.copy_(torch.tensor(c.lens))
        c.wide = torch.cat([x[b][done[b]:c.lens[b]] for b in range(2)])
        c.q = c.wide[:, :c.H]
        c.out = torch.full((c.T, c.H + 1, D), 7.0, dtype=torch.bfloat16, device="cuda")
        all_ids, c.ids = c.ids, [c.ids[b][:-(-c.lens[b] // P)] for b in range(2)]
        append(c, D, turns=turns, in_place=True)
        got = c.attend(window=window, sinks=sinks)
        capi.sync_check()
        c.check(got, *c.attended(window=window, sinks=sinks))
        c.ids = all_ids
        done = list(c.lens)
    for b in range(2):
        at = torch.arange(total[b], device="cuda")[:, None].expand(-1, D // 2)
        k, m = turned(x[b][:, whole.H:whole.H + Hkv], at, D, False, turns)
        v = x[b][:, whole.H + Hkv:].double()
        for i, want in enumerate((k, v)):
            held = whole.cached(i, b).transpose(0, 1)
            if not int8:
                assert bool(((held - want).abs() <= BF16 * want.abs() * 1.01 + 2 ** -22 * m).all())
                continue
            # half a step each time the page's factor grew, and once when the token came: a page's tokens came in at most 16 calls
            s = whole.scales[i][whole.ids[b], :Hkv].double().repeat_interleave(P, 0)[:total[b]]
            assert bool(((held - want).abs() <= s[..., None] * 0.51 * 16).all())
            assert float((held - want).abs().mean() / s.mean()) < 0.51
