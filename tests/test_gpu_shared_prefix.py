"""Attention of single tokens over shared pages against the definition in 64 bits, request by request."""
import ctypes

import numpy as np
import pytest
import torch

PAGE = 16
WIDE = False


@pytest.fixture(autouse=True, params=["narrow", "wide"])
def tables(request):
    """Every test twice: with block tables as wide as the requests are long, of which a small call reads every row by itself, and in bfloat16 with
    tables wide enough that what rows share is read once on the tensor cores."""
    global WIDE
    WIDE = request.param == "wide"


def make(runs, hq, hkv, d, dv=None, dtype=torch.bfloat16, seed=0, page=PAGE, sinks=False, spread=1.0, extra_width=0):
    """`runs`: [(rows' counts, shared positions)]; rows of a run share that many positions' pages. Pages in no order, a few unused ones among them."""
    dv = dv or d
    rng = np.random.default_rng(seed)
    counts = [c for cs, _ in runs for c in cs]
    width = max(1, -(-max(counts) // page)) + extra_width
    if WIDE and dtype == torch.bfloat16:
        width += -(-150_000_000 // (len(counts) * page * hkv * d * 4))
    table = np.full((len(counts), width), -1, np.int32)
    total = sum(shared // page + sum(max(0, -(-(c - shared) // page)) for c in cs) for cs, shared in runs) + 3
    pages = rng.permutation(total).astype(np.int32).tolist()
    ids, lens, r = [], [], 0
    for i, (cs, shared) in enumerate(runs):
        common = [pages.pop() for _ in range(shared // page)]
        for c in cs:
            n = -(-c // page)
            row = common[:n] + [pages.pop() for _ in range(max(0, n - len(common)))]
            table[r, :n] = row
            ids.append(i + 5)
            lens.append(shared)
            r += 1
    f = lambda *shape: torch.from_numpy(rng.normal(0.0, 1.0, shape).astype(np.float32)).cuda()
    on = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    return dict(q=(spread * f(len(counts), hq, d)).to(dtype), k=f(total, hkv, page, d).to(dtype), v=f(total, hkv, page, dv).to(dtype), table=on(table), count=on(counts),
                share_id=on(ids), share_len=on(lens), sinks=f(hq) if sinks else None, page=page, counts=counts)


def run(c, window=None, softcap=None, scale=None):
    from kapel_b200 import kernels as K

    return K.shared_prefix_attention(c["q"], c["k"], c["v"], c["table"], c["count"], c["share_id"], c["share_len"], c["page"], window,
                                     c["q"].shape[2] ** -0.5 if scale is None else scale, softcap, sinks=c["sinks"])


def plain(c, window=None, softcap=None, scale=None):
    """([rows, hq, dv], the sums of the weights times the values' sizes): the definition in 64 bits, out of each row's own block table."""
    q, table = c["q"].double().cpu().numpy(), c["table"].cpu().numpy()
    k, v = c["k"].double().cpu().numpy(), c["v"].double().cpu().numpy()
    rows, hq, d = q.shape
    hkv, dv, page = k.shape[1], v.shape[3], c["page"]
    scale = d ** -0.5 if scale is None else scale
    out, size = np.zeros((rows, hq, dv)), np.zeros((rows, hq, dv))
    for r in range(rows):
        count = c["counts"][r]
        at = np.arange(max(0, count - window) if window else 0, count)
        at = at[table[r, at // page] >= 0]
        if not at.size:
            continue
        for h in range(hq):
            keys, values = k[table[r, at // page], h // (hq // hkv), at % page], v[table[r, at // page], h // (hq // hkv), at % page]
            x = keys @ q[r, h] * scale
            if softcap:
                x = softcap * np.tanh(x / softcap)
            top = x.max() if c["sinks"] is None else max(x.max(), float(c["sinks"][h]))
            w = np.exp(x - top)
            total = w.sum() + (0.0 if c["sinks"] is None else np.exp(float(c["sinks"][h]) - top))
            out[r, h], size[r, h] = w @ values / total, w @ np.abs(values) / total
    return out, size


# float32: a score is a sum of d products, off by at most about d / 2 roundings of its terms' size; with the tests' queries and keys of standard
# deviation 1 and a scale of d^-1/2 that is well below 256 * 2^-24 * 8 = 1.2e-4 in the exponent at the very worst and a few 1e-6 as sums of
# rounded terms go; sums of weights and values add as much again. bfloat16: the weights that go into the products are rounded (2^-8 each
# of the values' sizes, at most), the result once more (2^-8); the scores' sums are 32-bit.
def check(c, **kw):
    got = run(c, **kw).double().cpu().numpy()
    want, size = plain(c, **kw)
    if c["q"].dtype == torch.float32:
        bound = 2e-5 * (size + 1e-3)
    else:
        bound = 2.0 ** -8 * size + 2.0 ** -8 * np.abs(want) + 1e-5
    worst = np.abs(got - want) - bound
    assert np.isfinite(got).all() and worst.max() <= 0, (np.unravel_index(worst.argmax(), worst.shape), np.abs(got - want).max(), want.shape)


HEADS = [(8, 4, 256), (16, 8, 128), (16, 4, 128), (8, 2, 64), (4, 4, 64), (12, 4, 96), (6, 2, 20), (16, 1, 128), (32, 1, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_heads_and_types(dtype, hq, hkv, d):
    check(make([([200, 161, 177, 193, 224], 160), ([40, 33], 32), ([7], 0)], hq, hkv, d, dtype=dtype, seed=d))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("runs", [
    [([1], 0)],                                              # one token, nothing before it
    [([16, 16], 16)],                                        # nothing of their own
    [([17, 17], 16)],
    [([0, 0, 5], 0)],                                        # rows that have seen nothing, as padding rows
    [([0, 40, 0], 32)],                                      # ... between rows that share
    [([64 + i for i in range(1, 40)], 64)],                  # more rows than a tile
    [([300] * 3, 128), ([300] * 3, 256), ([300] * 2, 16)],   # several prompts
    [([1000, 1003], 992), ([2], 0), ([5000], 0)],            # beside a long request of its own
    [([4097 + 31 * i for i in range(5)], 4096)],
    [([65], 64), ([65], 64)],                                # runs of one row
    [([30, 50, 70], 48)],                                    # a row that ends inside what is called shared
])
@pytest.mark.parametrize("hq,hkv,d", [(8, 4, 256), (16, 4, 128), (6, 2, 20)])
def test_lengths(dtype, runs, hq, hkv, d):
    check(make(runs, hq, hkv, d, dtype=dtype, seed=len(runs)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window", [1, 16, 50, 64, 100, 129, 1000])
@pytest.mark.parametrize("hq,hkv,d", [(8, 4, 256), (16, 4, 128)])
def test_windows(dtype, window, hq, hkv, d):
    runs = [([200, 161, 177, 193, 260, 400], 160), ([500], 0), ([321, 322], 320)]
    check(make(runs, hq, hkv, d, dtype=dtype, seed=window, sinks=window == 50), window=window, softcap=30.0 if window == 64 else None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("softcap,sinks", [(None, True), (50.0, False), (5.0, True), (0.5, False)])
@pytest.mark.parametrize("hq,hkv,d", [(8, 4, 256), (16, 2, 128), (4, 2, 64), (4, 2, 32)])
def test_soft_caps_and_sinks(dtype, softcap, sinks, hq, hkv, d):
    check(make([([300, 290, 271], 256), ([20], 0), ([0], 0)], hq, hkv, d, dtype=dtype, seed=3, sinks=sinks, spread=4.0), softcap=softcap)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,dv", [(64, 128), (128, 64), (20, 36), (96, 96)])
def test_values_of_another_size(dtype, d, dv):
    check(make([([100, 99, 130], 80), ([33], 0)], 8, 2, d, dv, dtype=dtype, seed=d, sinks=True))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("page", [16, 32, 64])
def test_pages_of_other_sizes(dtype, page):
    check(make([([300, 290, 271], 256), ([20], 0)], 8, 4, 128, dtype=dtype, page=page, extra_width=3))


@pytest.mark.gpu
def test_pages_of_an_odd_size():
    check(make([([50, 61], 40), ([20], 0)], 8, 4, 64, dtype=torch.float32, page=10))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_peaked_scores_of_both_signs(dtype):
    """Scores far apart: the running maximum moves, pieces fade to nothing; a negative scale turns the order around."""
    c = make([([700, 650, 641], 640), ([90], 0)], 8, 4, 128, dtype=dtype, seed=8, spread=12.0)
    for scale in (0.3, -0.3, 0.0):
        got = run(c, scale=scale).double().cpu().numpy()
        want, size = plain(c, scale=scale)
        # scores of up to about 0.3 * 12 * 128^0.5 * 4 = 163 carry 163 * 2^-24 * a few roundings into the exponent
        bound = (1e-4 if dtype == torch.float32 else 2.0 ** -7) * (size + 1e-3)
        assert np.isfinite(got).all() and (np.abs(got - want) <= bound).all(), (scale, np.abs(got - want).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", [(8, 4, 256), (16, 4, 128), (8, 2, 64), (6, 2, 20)])
def test_what_a_row_does_not_see_may_be_anything(dtype, hq, hkv, d):
    """NaN behind the last position of the last page, in pages nobody holds, below the window of a row that shares nothing; pages given back."""
    for window in (None, 70):
        c = make([([200, 161, 177], 160), ([131], 0), ([50], 0)], hq, hkv, d, dtype=dtype, seed=2)
        table, want = c["table"].cpu().numpy(), plain(c, window=window)
        seen = np.zeros(c["k"].shape[0] * PAGE, bool)
        for r, count in enumerate(c["counts"]):
            low = min((max(0, n - window) if window else 0) for n in c["counts"][:3]) if r < 3 else (max(0, count - window) if window else 0)
            at = np.arange(low, count)
            seen[table[r, at // PAGE] * PAGE + at % PAGE] = True
        for name, bad in (("k", float("nan")), ("v", float("nan")), ("v", float("inf"))):
            t = c[name].clone()
            lines = torch.from_numpy(np.flatnonzero(~seen)).cuda()
            t[lines // PAGE, :, lines % PAGE] = bad
            d2 = dict(c)
            d2[name] = t
            got = run(d2, window=window).double().cpu().numpy()
            bound = 2e-5 * (want[1] + 1e-3) if dtype == torch.float32 else 2.0 ** -8 * want[1] + 2.0 ** -8 * np.abs(want[0]) + 1e-5
            assert np.isfinite(got).all() and (np.abs(got - want[0]) <= bound).all(), (window, name, bad)
        if window:                                           # pages wholly below every window were given back
            d2, t2 = dict(c), table.copy()
            for r, count in enumerate(c["counts"]):
                low = min(max(0, n - window) for n in c["counts"][:3]) if r < 3 else max(0, count - window)
                t2[r, : low // PAGE] = -1
            d2["table"] = torch.from_numpy(t2).cuda()
            assert torch.equal(run(d2, window=window), run(c, window=window))
            for r, count in enumerate(c["counts"]):          # each its own, the longer one before the shorter one
                t2[r, : max(0, count - window) // PAGE] = -1
            d2["table"] = torch.from_numpy(t2).cuda()
            assert torch.equal(run(d2, window=window), run(c, window=window))


@pytest.mark.gpu
def test_shared_rows_are_the_rows_alone():
    """A group's rows give what each gives with nothing called shared, to the roundings of pieces joined in another order."""
    c = make([([700, 650, 641, 702], 640), ([90], 0)], 8, 4, 128, dtype=torch.float32, seed=8)
    alone = dict(c)
    alone["share_len"] = torch.zeros_like(c["share_len"])
    assert (run(c) - run(alone)).abs().max().item() < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_same_call_gives_the_same_bits(dtype):
    c = make([([700 + i for i in range(20)], 640), ([90], 0)], 8, 4, 128, dtype=dtype, seed=8)
    first = run(c)
    for _ in range(5):
        assert torch.equal(run(c), first)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_recorded_step_whose_lengths_change(dtype):
    """One recording, replayed with other lengths, groups and tables; a padding row at its end. Two recordings side by side."""
    shapes = [[([200, 161, 177], 160), ([40], 0), ([0], 0)], [([300, 290], 256), ([299, 257], 240), ([0], 0)], [([5], 0), ([6], 0), ([300], 0), ([1], 0), ([0], 0)]]
    cases = [make(s, 8, 4, 128, dtype=dtype, seed=i) for i, s in enumerate(shapes)]
    pages = max(c["k"].shape[0] for c in cases)
    width = max(c["table"].shape[1] for c in cases)
    for c in cases:
        grow = lambda t: torch.cat([t, torch.zeros((pages - t.shape[0], *t.shape[1:]), dtype=t.dtype, device="cuda")])
        c["k"], c["v"] = grow(c["k"]), grow(c["v"])
        c["table"] = torch.cat([c["table"], torch.full((5, width - c["table"].shape[1]), -1, dtype=torch.int32, device="cuda")], dim=1).contiguous()
    graphs = []
    for window in (None, 100):
        s = {n: cases[0][n].clone() for n in ("q", "k", "v", "table", "count", "share_id", "share_len")}
        s.update(page=PAGE, sinks=None)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(s, window=window)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(s, window=window)
        graphs.append((g, s, out, window))
    for c in cases + cases[:1]:
        for g, s, out, window in graphs:
            for n in ("q", "k", "v", "table", "count", "share_id", "share_len"):
                s[n].copy_(c[n])
            g.replay()
        for g, s, out, window in graphs:
            assert torch.equal(out, run(c, window=window))


@pytest.mark.gpu
def test_what_is_refused():
    from kapel_b200 import kernels as K

    c = make([([40, 41], 32)], 8, 4, 64)
    good = dict(q=c["q"], k_table=c["k"], v_table=c["v"], block_table=c["table"], row_count=c["count"], share_id=c["share_id"], share_len=c["share_len"],
                page_size=PAGE, window=None, scale=0.1, softcap=None)
    K.shared_prefix_attention(**good)
    for bad in (dict(q=c["q"].half()), dict(q=c["q"].float()), dict(q=c["q"][0]), dict(q=c["q"].transpose(0, 1)), dict(k_table=c["k"][:, :3].contiguous()), dict(page_size=8),
                dict(block_table=c["table"][:1]), dict(block_table=c["table"].long()), dict(row_count=c["count"][:1]), dict(share_id=c["share_id"].long()),
                dict(share_len=c["share_len"].cpu()), dict(window=-1), dict(softcap=-1.0), dict(sinks=torch.zeros(3, device="cuda")),
                dict(q=torch.zeros((2, 8, 300), dtype=torch.bfloat16, device="cuda"), k_table=torch.zeros((4, 4, PAGE, 300), dtype=torch.bfloat16, device="cuda"),
                     v_table=torch.zeros((4, 4, PAGE, 300), dtype=torch.bfloat16, device="cuda"))):
        with pytest.raises(K.KernelError):
            K.shared_prefix_attention(**{**good, **bad})
    e = K.shared_prefix_attention(**{**good, "q": c["q"][:0], "row_count": c["count"][:0], "share_id": c["share_id"][:0], "share_len": c["share_len"][:0]})
    assert e.shape == (0, 8, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [None, 1500])
@pytest.mark.parametrize("rows", [40, 70])                   # a step of few rows runs its two kernels side by side, a larger one does not
@pytest.mark.parametrize("hq,hkv,d", [(8, 4, 256), (16, 4, 128), (4, 2, 64)])
def test_many_units_a_block(hq, hkv, d, rows, window):
    check(make([([2400 + 1 + 13 * i % 200 for i in range(rows - 3)], 2400), ([800, 790], 752), ([1300], 0)], hq, hkv, d, seed=rows, spread=2.0), window=window, softcap=50.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shared_lengths_that_are_no_whole_pages(dtype):
    """Taken down to whole pages, to what the row has seen and to its block table; below a page, or negative, nothing is shared."""
    for shared, whole in ((175, 160), (15, 0), (-1, 0), (-2 ** 31, 0), (2 ** 31 - 1, None)):
        c = make([([200, 161, 177], 160), ([40], 0)], 8, 4, 128, dtype=dtype, seed=4)
        if whole is None:                                    # three rows with the same history, all of it shared
            c["count"][:3], c["counts"][:3] = 176, [176] * 3
            c["table"][:3] = c["table"][0].clone()
        c["share_len"][:3] = shared
        check(c)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", [(8, 4, 256), (16, 4, 128), (6, 2, 20)])
def test_own_pages_that_are_none_are_not_seen(dtype, hq, hkv, d):
    c = make([([200, 161, 177], 160), ([90], 0)], hq, hkv, d, dtype=dtype, seed=5)
    c["table"][0, 11] = -1
    c["table"][3, 1:3] = -7
    want, size = plain(c)
    c["table"][0, 11] = c["k"].shape[0]                      # beyond the tables
    c["table"][3, 2] = 2 ** 31 - 1
    got = run(c).double().cpu().numpy()
    bound = 2e-5 * (size + 1e-3) if dtype == torch.float32 else 2.0 ** -8 * size + 2.0 ** -8 * np.abs(want) + 1e-5
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.gpu
def test_one_page_many_times():
    """The same page at several places of a table, and in tables that share nothing."""
    c = make([([200, 161, 177], 160), ([90, 80], 0)], 8, 4, 128, seed=6)
    c["table"][:3, 3] = c["table"][0, 1].clone()
    c["table"][:3, 4] = c["table"][0, 1].clone()
    c["table"][4, 2:5] = c["table"][3, 0].clone()
    check(c)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_two_streams_at_once(dtype):
    cases = [make([([700 + 3 * i for i in range(12)], 640 - 64 * j), ([90 + j], 0)], 8, 4, 128, dtype=dtype, seed=j) for j in range(2)]
    want = [run(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[j].append(run(cases[j]))
    torch.cuda.synchronize()
    for j in range(2):
        for x in got[j]:
            assert torch.equal(x, want[j])


@pytest.mark.gpu
def test_the_most_rows():
    from kapel_b200 import kernels as K

    n = K.SHARED_PREFIX_ROWS
    check(make([([33 + i % 20 for i in range(n - 2)], 32), ([3, 70], 0)], 4, 2, 64, seed=1))
    with pytest.raises(K.KernelError):
        run(make([([33] * (n + 1), 32)], 4, 2, 64, seed=1))


def test_the_launcher_refuses_without_a_gpu():
    try:
        from kapel_b200 import kernels as K

        lib = K.library()
    except Exception as err:
        pytest.skip(f"the CUDA library cannot be built or loaded here: {err}")
    vp, i32, f32, i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_longlong

    def call(dtype=1, rows=4, hq=8, hkv=4, d=128, dv=128, page=16, width=64, pages=256, window=0, cap=0.0, scratch=4096, floats=1 << 40):
        a = vp(4096)
        return lib.kb_shared_attention(a, a, a, a, i32(dtype), a, a, a, a, *[i32(x) for x in (rows, hq, hkv, d, dv, page, width, pages, window)], f32(0.1), f32(cap),
                                       None, vp(scratch), i64(floats), None)

    for kw, word in ((dict(rows=513), "513 rows"), (dict(rows=-1), "-1 rows"), (dict(dtype=2), "dtype code 2"), (dict(hq=9), "9 heads over 4"), (dict(d=257), "of 257"),
                     (dict(dv=300), "/ 300"), (dict(hq=132, hkv=1), "132 heads"), (dict(page=0), "pages of 0"), (dict(width=0), "table width 0"), (dict(window=-2), "window -2"),
                     (dict(cap=-1.0), "soft cap -1"), (dict(scratch=0), "scratch"), (dict(floats=100), "scratch"), (dict(rows=512, hkv=1, width=1 << 24), "too many")):
        assert call(**kw) != 0
        assert word in lib.kb_last_error().decode(), lib.kb_last_error()
