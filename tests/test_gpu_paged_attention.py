"""GPU: attention over the paged cache (b200fc_paged_attention) against the formula in 64 bits."""
import math

import pytest
import torch

from mm_amx_b200 import capi
from paged_cases import Paged

pytestmark = pytest.mark.gpu


def run(c, **kw):
    got = c.attend(**kw)
    capi.sync_check()
    kw.pop("max_rows", None)
    c.check(got, *c.attended(**kw))


ONE_ROW = [
    ([0, 1, 2, 15, 16, 17, 31, 32, 33], 2, 2, 64, 16), ([63, 64, 65, 127, 128, 129, 500], 1, 4, 128, 16), ([1000, 3, 700], 8, 1, 128, 32),
    ([5000, 1, 0, 4999, 2500], 2, 8, 128, 64), ([300], 4, 16, 64, 128), ([77, 1030], 3, 7, 128, 128), ([40, 2000], 1, 32, 64, 16), ([1500], 2, 17, 128, 64),
    ([9000], 1, 1, 64, 64), ([i * 3 for i in range(300)], 1, 2, 64, 16),
]


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("lens,Hkv,G,D,page", ONE_ROW, ids=str)
def test_one_row(lens, Hkv, G, D, page, int8):
    """lengths around blocks and pages, none and one token, groups of any size; NaN behind every length"""
    run(Paged([1] * len(lens), lens, Hkv, G, D, page, int8, one_row=True))


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (17, 3), (100, 4), (64, 200), (1000, 16), (2 ** 31 - 1, 2 ** 31 - 1), (33, 2 ** 31 - 1)])
def test_one_row_with_window_and_sinks(window, sinks, D, int8):
    lens = [0, 1, 16, 17, 50, 99, 100, 101, 104, 105, 117, 400, 3000]
    run(Paged([1] * len(lens), lens, 2, 4, D, 32, int8, one_row=True), window=window, sinks=sinks)


FEW = [([3, 1, 0, 8, 5], [40, 1, 7, 8, 600], 2, 4, 128, 16), ([2, 2], [2, 1], 1, 1, 64, 16), ([6, 4, 5], [4096, 3000, 100], 4, 8, 128, 16), ([12, 1], [500, 200], 1, 16, 64, 64),
       ([16] * 20, [33 * i + 16 for i in range(20)], 2, 1, 64, 32), ([7, 9], [1300, 9], 2, 5, 128, 128)]


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("rows,lens,Hkv,G,D,page", FEW, ids=str)
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 2)])
def test_few_rows(rows, lens, Hkv, G, D, page, int8, window, sinks):
    run(Paged(rows, lens, Hkv, G, D, page, int8, extra=3, row0=2), window=window, sinks=sinks)


PROMPTS = [([100], [100], 2, 2, 64, 16), ([128, 256, 129], [128, 256, 129], 1, 4, 128, 32), ([257, 1, 0, 65], [600, 400, 5, 65], 2, 3, 128, 64),
           ([513], [2000], 1, 8, 64, 128), ([300, 40], [280, 0], 2, 1, 128, 16), ([700, 1500], [700, 2047], 1, 2, 128, 64), ([31, 33, 500], [1031, 33, 777], 2, 7, 64, 16),
           ([127, 128, 129, 1], [127, 400, 129, 900], 2, 1, 64, 32), ([1000, 200], [3000, 200], 1, 3, 64, 128)]


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("rows,lens,Hkv,G,D,page", PROMPTS, ids=str)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (130, 5), (500, 300), (2 ** 31 - 1, 2)])
def test_prompts(rows, lens, Hkv, G, D, page, int8, window, sinks):
    """prompts and chunks of prompts, among them rows that stand for no token; rows of no sequence before and behind them"""
    run(Paged(rows, lens, Hkv, G, D, page, int8, extra=5, row0=1), window=window, sinks=sinks)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("n,Hkv,G", [(32, 2, 4), (33, 2, 4), (64, 2, 4), (65, 2, 4), (100, 1, 1), (1000, 1, 20)])
def test_prompts_of_many_sequences(n, Hkv, G, int8):
    """more sequences than are put in order by what they see, and than a block looks at together; decode rows and prompts side by side, some without rows"""
    rows = [0 if i % 11 == 5 else (1 if i % 3 else 20 + i % 40) for i in range(n)]
    run(Paged(rows, [r + (i * 37) % 200 for i, r in enumerate(rows)], Hkv, G, 64, 16, int8, extra=1))


@pytest.mark.parametrize("rows,lens,Hkv,G,D", [([2000], [2000], 1, 1, 128), ([300], [9000], 1, 2, 64), ([40], [20000], 2, 4, 128), ([129, 60], [5000, 7000], 1, 2, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (3000, 40)])
def test_long_contexts(rows, lens, Hkv, G, D, window, sinks):
    """tiles whose blocks several CTAs share, and rings that go round many times"""
    run(Paged(rows, lens, Hkv, G, D, 64), window=window, sinks=sinks)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("layout", ["places", "padded"])
@pytest.mark.parametrize("rows,lens", [([1, 1, 1], [300, 17, 1]), ([200, 3], [330, 170])])
def test_layouts(layout, rows, lens, int8):
    run(Paged(rows, lens, 2, 4, 128, 32, int8, layout=layout), window=90, sinks=3)
    run(Paged(rows, lens, 3, 2, 64, 16, int8, layout=layout))


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("rows,lens", [([1, 1], [2000, 150]), ([140, 5], [900, 70])])
@pytest.mark.parametrize("scale", [0.0, 1.0, -0.5, 4.0])
def test_scales_of_the_scores(rows, lens, int8, scale):
    """sharply peaked weights, equal weights, and weights that favour the smallest products.  Scores of up to |s| = 4 * 60 are off by 240 * 2^-24 * 8 at most"""
    run(Paged(rows, lens, 2, 4, 128, 16, int8), scale=scale)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("rows,lens,window", [([1, 1], [2000, 150], 0), ([140, 5, 300], [900, 70, 300], 0), ([400], [900], 70)])
def test_rising_scores(rows, lens, window, int8):
    """keys that grow with their place: the running maximum moves again and again"""
    c = Paged(rows, lens, 1, 4, 128, 16, int8)
    for b, ids in enumerate(c.ids):
        for j, pg in enumerate(ids):
            if int8:
                c.scales[0][pg] *= 0.05 + 0.3 * j
            else:
                c.pool[0][pg] *= 0.05 + 0.3 * j
    run(c, window=window)


@pytest.mark.parametrize("rows,lens,window,sinks", [([1, 1], [400, 150], 0, 0), ([1, 1], [400, 150], 100, 5), ([9, 3], [300, 77], 30, 4), ([200, 140], [330, 140], 0, 0),
                                                    ([300, 100], [700, 120], 50, 20),
                                                    ([40], [6000], 0, 0), ([6, 2], [3000, 1000], 0, 0)])
def test_values_that_are_no_numbers(rows, lens, window, sinks):
    """a NaN or an infinity in v reaches the rows that see its token, and no other row of the call; one in an invisible key reaches nobody"""
    c = Paged(rows, lens, 2, 4, 64, 16)
    for b, n in enumerate(lens):
        for at, what in ((n - 1, float("nan")), (n - 40, float("inf")), (n // 3, float("nan")), (30, float("-inf"))):
            if at < 0:
                continue
            c.pool[1][c.ids[b][at // 16], b % 2, at % 16, 5 + b] = what
        # a key that the last row alone sees, and one in front of every window
        if rows[b] > 1:
            c.pool[0][c.ids[b][(n - 1) // 16], 1, (n - 1) % 16, 3] = float("nan")
        low = n - rows[b] - window
        if window and low > sinks:
            c.pool[0][c.ids[b][low // 16], 0, low % 16] = float("nan")
    run(c, window=window, sinks=sinks)


@pytest.mark.parametrize("rows,lens", [([1, 1], [400, 150]), ([3, 4], [300, 77]), ([200, 140], [330, 140]), ([40, 30], [6000, 100])])
def test_rows_of_q_that_are_no_numbers(rows, lens):
    """a NaN in q stays with its row and head"""
    c = Paged(rows, lens, 2, 4, 128, 16)
    hit = [(0, 1), (rows[0] - 1, 6), (c.T - 1, 2)]
    want, mag = c.attended()
    for r, h in hit:
        c.q[r, h, 77] = float("nan")
        want[r, h] = float("nan")
    got = c.attend()
    capi.sync_check()
    c.check(got, want, mag)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows", [[1, 1], [3, 5], [300, 40]], ids=str)
def test_kv_heads_that_lie_on_one_another(rows, D, int8):
    """a head stride of 0 (which no tensor map has)"""
    c = Paged(rows, [700, 333], 2, 4, D, 32, int8)
    c.pool = [t[:, :1].expand(-1, 2, -1, -1) for t in c.pool]
    assert c.cache().head_stride == 0
    run(c)
    run(c, window=100, sinks=40)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("rows", [[1, 1, 1], [2, 3, 1], [60, 200, 1]], ids=str)
def test_sequences_that_share_their_first_pages(rows, int8):
    """what several sequences begin with stands in the cache once"""
    c = Paged(rows, [320, 300, 129], 2, 4, 64, 16, int8)
    for b in (1, 2):
        c.ids[b][:5] = c.ids[0][:5]
        c.table[b, :5] = c.table[0, :5]
    run(c)
    run(c, window=250, sinks=3)


def test_pages_that_no_row_sees_are_not_read():
    """pages behind the window may have been given back: their entries name other pages, or none"""
    for rows, lens in (([1, 1], [1000, 300]), ([40], [900])):
        c = Paged(rows, lens, 1, 4, 128, 16)
        ref = c.attended(window=64, sinks=4)
        for b, n in enumerate(lens):
            first = (n - rows[b] - 64 + 1) // 16
            for j in range(1, first):
                c.table[b, j] = -5
                for i in range(2):
                    c.pool[i][c.ids[b][j]] = float("nan")
        got = c.attend(window=64, sinks=4)
        capi.sync_check()
        c.check(got, *ref)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("rows,lens", [([1, 1, 1], [100, 200, 40]), ([150, 40, 2], [200, 200, 40])])
def test_pages_outside_the_pool_are_reported_and_left_out(rows, lens, int8):
    c = Paged(rows, lens, 2, 2, 64, 16, int8)
    for entry in (c.pages, -1, 2 ** 31 - 1):
        c.table[1, 3] = entry
        c.attend()
        with pytest.raises(capi.B200FCError) as e:
            capi.sync_check()
        assert e.value.code == capi.ERR_INVALID and "paged" in str(e.value)
        capi.sync_check()                            # reported once
        ref, mag = c.attended()
        got = c.out[:, :c.H].double()
        for b in (0, 2):                             # the others are not touched by it
            r = slice(c.starts[b], c.starts[b + 1])
            assert float(((got - ref).abs() - (2.0 ** -8 * 1.01 * (mag + ref.abs()) + 3e-4 * mag))[r].max()) <= 0
        assert bool(torch.isfinite(got).all())


@pytest.mark.parametrize("rows,max_rows", [([1, 1, 1], 1), ([20, 150, 30], 150)])
def test_numbers_outside_their_buffers_are_reported_and_left_out(rows, max_rows):
    lens = [r + 50 for r in rows]
    c = Paged(rows, lens, 2, 2, 64, 16)
    ref, mag = c.attended()
    keep = c.row_start.clone()

    def broken():
        c.out.fill_(7.0)
        c.attend(max_rows=max_rows)
        with pytest.raises(capi.B200FCError) as e:
            capi.sync_check()
        assert e.value.code == capi.ERR_INVALID
        got = c.out[:, :c.H].double()
        r = slice(c.starts[0], c.starts[1])
        assert float(((got - ref).abs() - (2.0 ** -8 * 1.01 * (mag + ref.abs()) + 3e-4 * mag))[r].max()) <= 0
        return got

    for n in (-1, 2 ** 31 - 1, c.table.shape[1] * 16 + 1):
        c.seq_lens[2] = n
        assert bool((broken()[c.starts[2]:c.starts[3]] == 7.0).all())
    c.seq_lens[2] = lens[2]
    for last in (c.T + 1, -1, 2 ** 31 - 1, -2 ** 31):
        c.row_start[3] = last
        assert bool((broken()[c.starts[2]:c.starts[3]] == 7.0).all())
    c.row_start.copy_(keep)
    if max_rows > 1:
        max_rows = 149
        assert bool((broken()[c.starts[1]:c.starts[2]] == 7.0).all())


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("rows,lens", [([1, 1], [40, 600]), ([130, 20], [200, 90])])
def test_places_past_32_bits(rows, lens, int8):
    """pages, heads and tokens whose offsets pass 2^31 and 2^32 bytes"""
    c = Paged(rows, lens, 2, 2, 64, 16, int8)
    es = 1 if int8 else 2
    ref = c.attended()
    # pages 150 MB apart and heads 75 MB: more than 50 pages reach past 7 GB
    stride = 150_000_000 // 16 * 16
    need = c.pages * stride + 4096
    big = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in range(2)]
    for i in range(2):
        view = big[i].view(c.pool[i].dtype).as_strided(tuple(c.pool[i].shape), (stride // es, stride // 2 // es, 64, 1))
        view.copy_(c.pool[i])
        c.pool[i] = view
    got = c.attend()
    capi.sync_check()
    c.check(got, *ref)


@pytest.mark.parametrize("rows,lens,Hkv", [([1] * 3, [5000, 100, 3000], 2), ([6, 2], [3000, 50], 2), ([200, 100], [900, 100], 1)])
def test_captured_calls_keep_their_own_workspaces(rows, lens, Hkv):
    """two graphs captured on one stream, a larger call between their replays, new lengths and pages at replay"""
    cs = [Paged(rows, lens, Hkv, 4, 128, 16, seed=i) for i in range(2)]
    other = Paged([r for r in rows] * 4, [n for n in lens] * 4, Hkv, 8, 128, 16)
    s = torch.cuda.Stream()
    graphs = []
    for c in cs:
        c.attend()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            c.attend(stream=s.cuda_stream)
        graphs.append(graph)
    for turn in range(2):
        for c, graph in zip(cs, graphs):
            c.out.fill_(7.0)
            if turn:                                # a shorter first sequence, its pages the other way round
                n = c.lens[0] = lens[0] // 2 + rows[0]
                c.seq_lens[0] = n
                c.ids[0] = c.ids[0][:-(-n // 16)][::-1]
                c.table[0, :len(c.ids[0])] = torch.tensor(c.ids[0], dtype=torch.int32, device="cuda")
            other.attend(stream=s.cuda_stream)
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for c in cs:
            c.check(c.out[:, :c.H], *c.attended())
    capi.sync_check()


def test_calls_on_two_streams_at_once():
    cs = [Paged([1] * 4, [4000, 100, 2000, 3000], 2, 4, 128, 16, seed=1), Paged([250, 5], [900, 1000], 2, 4, 128, 16, seed=2)]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s in zip(cs, streams):
            c.attend(stream=s.cuda_stream)
    torch.cuda.synchronize()
    capi.sync_check()
    for c in cs:
        c.check(c.out[:, :c.H], *c.attended())


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("rows,lens", [([1] * 5, [3000, 10, 500, 7000, 1]), ([4, 5], [3000, 100]), ([300, 70], [900, 70])])
def test_the_same_call_gives_the_same_bits(rows, lens, int8):
    c = Paged(rows, lens, 2, 4, 128, 64, int8)
    first = c.attend().clone()
    for _ in range(5):
        assert torch.equal(c.attend(), first)
    capi.sync_check()


@pytest.mark.parametrize("D,window", [(64, 0), (128, 0), (64, 9)])
def test_pairs_with_and_without_odd_values_one_after_another(D, window):
    """single blocks handle several (sequence, kv head) pairs in turn: a NaN in one pair's newest values neither reaches the next pair nor leaves a row out"""
    n = 500
    c = Paged([2 + b % 3 for b in range(n)], [20 + b * 7 % 50 for b in range(n)], 4, 2, D, 16)
    for b in range(0, n, 2):
        at = c.lens[b] - 1
        c.pool[1][c.ids[b][at // 16], b // 2 % 4, at % 16, 9] = float("nan")
    ref = c.attended(window=window)
    for _ in range(5):
        c.out.fill_(7.0)
        got = c.attend(window=window)
        capi.sync_check()
        c.check(got, *ref)


@pytest.mark.parametrize("how", ["infinite", "overflow", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows,lens,window,sinks", [([1, 1], [400, 150], 0, 0), ([1, 1, 1], [5000, 3, 700], 0, 0), ([1, 1], [3000, 150], 100, 40), ([3, 2], [300, 77], 0, 0),
                                                    ([8, 5], [3000, 500], 90, 20), ([200, 20], [330, 70], 0, 0), ([300, 40], [900, 300], 100, 30), ([40], [6000], 0, 0)])
def test_scores_of_minus_infinity(rows, lens, window, sinks, D, how):
    """visible keys whose score is -inf (an infinity in k, or products beyond fp32) weigh nothing, wherever they stand: all in front of the rows' own places, and every third
    block of 16 tokens from there on.  (Each row sees a token with another score: its sequence's first row's, or one of the two blocks between.)"""
    c = Paged(rows, lens, 2, 4, D, 16, how == "int8")
    big = 2.0 ** 127
    c.q[..., 3] = 1.0 if how == "infinite" else big
    for b, n in enumerate(lens):
        for j in range(n):
            low = j < n - rows[b] or j // 16 % 3 == 0 and j > n - rows[b]
            c.pool[0][c.ids[b][j // 16], :, j % 16, 3] = 0 if not low else {"infinite": float("-inf"), "overflow": -big, "int8": -127}[how]
    run(c, window=window, sinks=sinks)


@pytest.mark.parametrize("rows,lens", [([1, 1], [400, 3]), ([4, 2], [300, 7]), ([200, 20], [330, 70]), ([40], [6000])])
def test_rows_whose_every_score_is_minus_infinity(rows, lens):
    c = Paged(rows, lens, 2, 4, 128, 16)
    c.q[..., 3] = 1.0
    for b, n in enumerate(lens):
        c.pool[0][c.ids[b], :, :, 3] = float("-inf")
    got = c.attend()
    capi.sync_check()
    assert bool((got == 0).all())


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("n,rows", [(700, 5), (20, 9), (300, 1)])
def test_every_sequence_outside_its_buffers_is_reported(n, rows, int8):
    """wherever it stands among the call's sequences, with rows or without; the others get their results"""
    rows = [0 if b % 9 == 7 else rows for b in range(n)]
    c = Paged(rows, [9 + b % 7 for b in range(n)], 1, 8, 64, 16, int8)
    ref, mag = c.attended()
    starts, lens = c.row_start.clone(), c.seq_lens.clone()

    def broken(harmed):
        c.out.fill_(7.0)
        c.attend()
        with pytest.raises(capi.B200FCError) as e:
            capi.sync_check()
        assert e.value.code == capi.ERR_INVALID
        over = (c.out[:, :c.H].double() - ref).abs() - (2.0 ** -8 * 1.01 * (mag + ref.abs()) + 3e-4 * mag)
        unharmed = torch.ones(c.T, dtype=torch.bool, device="cuda")
        for b in harmed:
            unharmed[c.starts[b]:c.starts[b + 1]] = False
            assert bool((c.out[c.starts[b]:c.starts[b + 1]] == 7.0).all())
        assert float(over[unharmed].max()) <= 0
        c.row_start.copy_(starts); c.seq_lens.copy_(lens)

    for b in {0, 7, n // 3, n // 2 + 1, 63 % n, 64 % n, 256 % n, 691 % n, n - 1}:
        for length in (-1, 2 ** 31 - 1, c.table.shape[1] * 16 + 1):
            c.seq_lens[b] = length
            broken([b])
    c.row_start[n] = c.T + 1
    broken([n - 1])
    c.row_start[n - 5] = -1
    broken([n - 6, n - 5])


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("rows,lens", [([1, 1, 1], [9000, 3, 700]), ([3, 2], [3000, 77]), ([200, 140], [330, 700]), ([40], [20000])])
@pytest.mark.parametrize("D", [64, 128])
def test_the_largest_values(D, rows, lens, int8):
    """|v| times the visible tokens just below 2^119, with scores behind the first 128 tokens that are 7.9 / log2(e) higher, so that weights reach nearly 2^8.  (The sums
    of p v are then below 2^127 (1 + 2^-7): finite.)"""
    c = Paged(rows, lens, 2, 4, D, 16, int8, std=0.02)
    c.q[..., 3] = 8.0
    size = 0.99 * 2.0 ** 119 / max(lens)
    sign = torch.where(torch.rand(2, 1, D, generator=c.g, device="cuda") < 0.5, -1.0, 1.0)
    for ids in c.ids:
        for j, pg in enumerate(ids):
            if int8:
                c.pool[1][pg] = (127 * sign).to(torch.int8)
                c.scales[0][pg, :2], c.scales[1][pg, :2] = 0.7 / 127, size / 127
                c.pool[0][pg, ..., 3] = 0 if j < 8 else 124
                c.pool[0][pg, ..., :3] = 0
                c.pool[0][pg, ..., 4:] = 0
            else:
                c.pool[1][pg] = (size * sign).to(torch.bfloat16)
                c.pool[0][pg, ..., 3] = 0.0 if j < 8 else 7.9 / 8 * math.log(2)
    run(c, scale=1.0)
    run(c, scale=1.0, window=100, sinks=4)


@pytest.mark.parametrize("rows,lens", [([1, 1], [400, 150]), ([3, 2], [300, 77]), ([200, 20], [330, 70])])
def test_the_largest_factors_of_keys(rows, lens):
    """k_scale and k_scale * scale just below 2^121, met by rows of q so small that the scores are ordinary (four components of +- 2^-121 against integers of 0 and +- 32:
    sums of up to four times 32, so that all products and scores are normal numbers of fp32), every other row all zeros"""
    c = Paged(rows, lens, 2, 4, 64, 16, True)
    c.scales[0][:, :2].mul_(0.99 * 2.0 ** 121 / float(c.scales[0][c.ids[0] + c.ids[1], :2].max()))
    c.pool[0].copy_((c.pool[0].float() / 64).round().clamp(-1, 1) * 32)
    c.q.copy_(torch.sign(c.q) * 2.0 ** -121 * (torch.arange(64, device="cuda") % 16 == 5))
    c.q[1::2] = 0.0
    run(c)
    run(c, scale=1.0)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_prompts_and_single_tokens_in_two_calls(int8):
    """the sequences of a mixed batch with prompts first: one call for them, one without row_start for the others, on parts of the same buffers"""
    c = Paged([150, 40, 1, 1, 1], [400, 40, 900, 1, 77], 2, 4, 128, 32, int8)
    ref = c.attended()
    for first, count, row, rows, one_row in ((0, 2, 0, 190, False), (2, 3, 190, 3, True)):
        cache = c.cache(B=count, page_table=c.table[first:].data_ptr(), seq_lens=c.seq_lens[first:].data_ptr())
        q, out = c.q[row:], c.out[row:]
        capi.paged_attention(capi.PagedAttention(
            cache=capi.pointer(cache), T=rows, max_rows=1 if one_row else 150, H=c.H, row_start=None if one_row else c.row_start.data_ptr(), q=q.data_ptr(),
            q_row_stride=q.stride(0) * 2, q_head_stride=q.stride(1) * 2, out=out.data_ptr(), out_row_stride=out.stride(0) * 2, out_head_stride=out.stride(1) * 2,
            scale=c.D ** -0.5))
    capi.sync_check()
    c.check(c.out[:, :c.H], *ref)
