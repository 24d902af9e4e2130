"""The 8-bit paged cache against its oracle in float64: block tables, append, attention of new tokens over the cache."""
import numpy as np
import pytest
import torch

from oracle import cache_oracle as orc

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def ints(x, device="cuda"):
    return torch.tensor(np.ascontiguousarray(x), dtype=torch.int32, device=device)


def row_of(dim):
    return 32 if dim <= 32 else 64 if dim <= 64 else 128


# -------------------------------------------------------------------------------------------------------------- block tables
def blocks_case(rng, R, page, width, spare, most):
    lengths = rng.integers(0, width * page + 1, R)
    new = np.array([rng.integers(-t, min(most, width * page - t) + 1) for t in lengths])
    new[rng.random(R) < 0.2] = 0
    held = -(-lengths // page)
    pages = int(held.sum()) + spare
    order = rng.permutation(pages)
    tables = np.full((R, width), -7)
    at = 0
    for r in range(R):
        tables[r, :held[r]] = order[at:at + held[r]]
        at += held[r]
    free = np.full(pages, -9)
    free[:pages - at] = order[at:]
    return lengths, new, tables, free, pages - at


def run_blocks(lengths, new, tables, free, count, page, tokens):
    from stickbreaking_attention_b200 import sb_cache_blocks
    t, f = ints(tables), ints(free)
    s = sb_cache_blocks(ints(lengths), ints(new), t, f, ints([count]), page, tokens)
    return [x.cpu().numpy() for x in (s.lengths, s.free_count, s.ends, s.slots, s.pieces, t, f)]


@pytest.mark.parametrize("R, page, width, most", [(1, 16, 3, 20), (1, 128, 1, 5), (5, 16, 4, 1), (40, 32, 6, 70), (256, 64, 20, 3), (257, 16, 5, 90), (1000, 16, 7, 40)])
@pytest.mark.parametrize("seed", [0, 1])
def test_blocks(R, page, width, most, seed):
    rng = np.random.default_rng(seed)
    case = blocks_case(rng, R, page, width, 5 * R * (most // page + 2), most)
    tokens = int(np.maximum(case[1], 0).sum()) + 3 * seed
    want = orc.blocks(*case, page, tokens)
    assert want is not None
    for got, ref in zip(run_blocks(*case, page, tokens), want):
        assert np.array_equal(got, np.atleast_1d(ref))


def test_blocks_pages_given_back_are_taken_again():
    """No free page but those that other requests give up in the same step, to the last one."""
    page, tables = 16, np.array([[0, 1, 2, -1], [3, 4, -1, -1], [5, -1, -1, -1]])
    case = (np.array([40, 17, 16]), np.array([-40, -2, 48]), tables, np.full(6, -1), 0)
    want = orc.blocks(*case, page, 48)
    got = run_blocks(*case, page, 48)
    for g, w in zip(got, want):
        assert np.array_equal(g, np.atleast_1d(w))
    assert got[1][0] == 1 and list(got[5][2]) == [5, 4, 2, 1]


def test_blocks_is_repeatable_until_its_lengths_are_taken_over():
    from stickbreaking_attention_b200 import sb_cache_blocks
    rng = np.random.default_rng(3)
    lengths, new, tables, free, count = blocks_case(rng, 33, 16, 5, 60, 40)
    t, f, args = ints(tables), ints(free), (ints(lengths), ints(new))
    first = [x.clone() for x in sb_cache_blocks(*args, t, f, ints([count]), 16, 2000)] + [t.clone(), f.clone()]
    again = list(sb_cache_blocks(*args, t, f, ints([count]), 16, 2000)) + [t, f]
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("what", ["pages", "tokens", "long", "below", "length", "count"])
def test_blocks_refused_on_the_device(what, monkeypatch):
    from stickbreaking_attention_b200 import check_status, sb_cache_blocks
    monkeypatch.setenv("SBATTN_CHECK_STATUS", "0")
    page, tables, free = 16, ints([[0, 1, -1], [2, -1, -1]]), ints([3, 4, 5, -1])
    lengths, new, count, tokens = [20, 3], [5, 30], 3, 64
    if what == "pages":
        count = 0
    elif what == "tokens":
        tokens = 34
    elif what == "long":
        new = [5, 46]
    elif what == "below":
        new = [-21, 1]
    elif what == "length":
        lengths = [20, -1]
    else:
        count = 5
    t, f = tables.clone(), free.clone()
    s = sb_cache_blocks(ints(lengths), ints(new), t, f, ints([count]), page, tokens)
    with pytest.raises(ValueError, match="free pages" if what == "pages" else "rejected"):
        check_status()
    assert torch.equal(t, tables) and torch.equal(f, free) and s.lengths.tolist() == lengths and s.free_count.tolist() == [count]
    assert s.ends.tolist() == [0, 0] and (s.slots == -1).all() and (s.pieces[:, 0] == -1).all()
    assert check_status() == 0


def test_blocks_without_requests_or_tokens():
    from stickbreaking_attention_b200 import sb_cache_blocks
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    s = sb_cache_blocks(none, none, none.view(0, 4), none, ints([0]), 16, 3)
    assert s.slots.tolist() == [-1] * 3 and s.free_count.tolist() == [0] and s.pieces.shape == (0, 4)
    s = sb_cache_blocks(ints([5]), ints([0]), ints([[2, -1]]), ints([0, 1, 3]), ints([3]), 16, 0)
    assert s.slots.shape == (0,) and s.lengths.tolist() == [5] and s.ends.tolist() == [0]


def test_blocks_strided_table():
    rng = np.random.default_rng(5)
    lengths, new, tables, free, count = blocks_case(rng, 9, 16, 4, 40, 30)
    from stickbreaking_attention_b200 import sb_cache_blocks
    wide = torch.full((9, 11), -3, dtype=torch.int32, device="cuda")
    wide[:, 2:6] = ints(tables)
    f = ints(free)
    sb_cache_blocks(ints(lengths), ints(new), wide[:, 2:6], f, ints([count]), 16, 500)
    want = orc.blocks(lengths, new, tables, free, count, 16, 500)
    assert np.array_equal(wide[:, 2:6].cpu().numpy(), want[5]) and (wide[:, :2] == -3).all() and (wide[:, 6:] == -3).all()


# -------------------------------------------------------------------------------------------------------------------- append
def filled_cache(rng, pages, heads, page, dim, halves=False):
    """A cache with something in every page (other requests' tokens, leftovers), as numpy codes and scales and as tensors."""
    from stickbreaking_attention_b200 import SbCache
    row = row_of(dim)
    codes = [rng.integers(0, 256, (pages, heads, page, row)).astype(np.uint8) for _ in range(2)]
    scales = [(2.0 ** rng.integers(-9, -3, (pages, heads))).astype(np.float32) for _ in range(2)]
    for c in codes:
        c[c & 127 == 127] = 0
        c[..., dim:] = 0
    if halves:  # keys and values of a page beside one another
        both = torch.tensor(np.stack(codes, 1), device="cuda").view(torch.float8_e4m3fn)
        sc = torch.tensor(np.stack(scales, 1), device="cuda")
        return codes, scales, SbCache(both[:, 0], both[:, 1], sc[:, 0], sc[:, 1])
    t = [torch.tensor(c, device="cuda").view(torch.float8_e4m3fn) for c in codes] + [torch.tensor(s, device="cuda") for s in scales]
    return codes, scales, SbCache(*t)


def check_append(rng, x, codes, scales, cache, pieces):
    from stickbreaking_attention_b200 import sb_cache_append
    sb_cache_append(x[0], x[1], cache, ints(pieces))
    for new, c, s, gc, gs in zip(x, codes, scales, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        wc, ws = orc.append(new.double().cpu().numpy(), c, s, pieces)
        assert np.array_equal(gs.cpu().numpy(), ws.astype(np.float32))
        assert np.array_equal(gc.contiguous().view(torch.uint8).cpu().numpy(), wc)


def random_pieces(rng, pages, page, n, tokens_per, shuffle=True):
    pieces, row = [], 0
    for p in rng.permutation(pages)[:n]:
        new = int(rng.integers(1, min(page, tokens_per) + 1))
        old = int(rng.integers(0, page - new + 1)) if rng.random() < 0.7 else 0
        pieces.append((int(p), row, old, new))
        row += new
    return np.array(pieces + [(-1, 0, 0, 0)] * 2), row


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim, page", [(128, 64), (64, 16), (50, 32), (7, 16), (32, 128), (100, 128), (1, 16), (128, 16)])
def test_append(dtype, dim, page):
    rng = np.random.default_rng(dim + page)
    codes, scales, cache = filled_cache(rng, 9, 3, page, dim)
    pieces, rows = random_pieces(rng, 9, page, 6, 1000)
    size = np.exp(rng.normal(0, 2, (3, rows, 1)))
    x = [torch.tensor(rng.normal(0, 1, (3, rows, dim)) * size, device="cuda").to(DTYPES[dtype]) for _ in range(2)]
    check_append(rng, x, codes, scales, cache, pieces)


@pytest.mark.parametrize("halves", [False, True])
def test_append_single_tokens(halves):
    """One token per page, at every place of it, louder and softer than what is there."""
    rng = np.random.default_rng(11)
    codes, scales, cache = filled_cache(rng, 40, 2, 16, 64, halves)
    pieces = np.array([(p, i, i % 16, 1) for i, p in enumerate(rng.permutation(40)[:33])])
    x = [torch.tensor(rng.normal(0, 1, (2, 33, 64)) * 10.0 ** rng.integers(-4, 4, (2, 33, 1)), device="cuda").bfloat16() for _ in range(2)]
    check_append(rng, x, codes, scales, cache, pieces)


@pytest.mark.parametrize("values", ["zeros", "inf", "nan", "all-nan", "huge", "tiny", "subnormal", "border", "minus-zero"])
def test_append_values(values):
    rng = np.random.default_rng(2)
    codes, scales, cache = filled_cache(rng, 3, 2, 16, 32)
    x = rng.normal(0, 1, (2, 9, 32)).astype(np.float32)
    if values == "zeros":
        x[:] = 0
    elif values == "inf":
        x[0, 3, 5], x[1, 1, 1] = np.inf, -np.inf
    elif values == "nan":
        x[0, 3, 5] = np.nan
    elif values == "all-nan":
        x[:] = np.nan
    elif values == "huge":
        x[0, 2, 2], x[1, 0, 0] = 3.4028234e38, -3.3e38
    elif values == "tiny":
        x *= 1e-36
    elif values == "subnormal":
        x *= 1e-40
    elif values == "border":  # just at, below and above 448 of a scale, and halves of a step
        x[0] = np.resize(np.array([448, 447.99997, 232, 8.5, 9.5, 0.0009765625], np.float32), (9, 32))
        x[1] = np.resize(np.array([448.00003, 2 ** -10, 3 * 2 ** -10, 17, 19], np.float32), (9, 32))
    else:
        x[:] = -0.0
    t = torch.tensor(x, device="cuda")
    check_append(rng, [t, t.flip(0).contiguous()], codes, scales, cache, np.array([(2, 0, 0, 4), (0, 4, 11, 5)]))


def test_append_strides():
    """Token-major projections, an inner stride, a broadcast head."""
    rng = np.random.default_rng(4)
    for make in (lambda a: a.permute(1, 0, 2).contiguous().permute(1, 0, 2), lambda a: torch.stack([a, a], -1)[..., 0], lambda a: a[:1].expand(3, -1, -1),
                 lambda a: a.transpose(1, 2).contiguous().transpose(1, 2)):
        codes, scales, cache = filled_cache(rng, 4, 3, 32, 40)
        pieces, rows = random_pieces(rng, 4, 32, 3, 30)
        x = [make(torch.tensor(rng.normal(0, 1, (3, rows, 40)), device="cuda").half()) for _ in range(2)]
        check_append(rng, x, codes, scales, cache, pieces)


@pytest.mark.parametrize("piece", [(4, 0, 0, 1), (0, 0, 16, 1), (0, 0, -1, 1), (0, 0, 0, 0), (0, 0, 0, 17), (0, 5, 0, 2), (0, -1, 0, 1), (1 << 30, 0, 0, 1), (0, 0, 0, -5),
                                   (0, 2147483647, 0, 1), (0, 0, 2147483647, 1), (0, 0, 0, 2147483647)])
def test_append_bad_pieces(piece, monkeypatch):
    """Pieces that do not fit the cache or the tokens are left out and reported; the others are done."""
    from stickbreaking_attention_b200 import check_status, sb_cache_append
    monkeypatch.setenv("SBATTN_CHECK_STATUS", "0")
    rng = np.random.default_rng(6)
    codes, scales, cache = filled_cache(rng, 4, 2, 16, 32)
    x = torch.tensor(rng.normal(0, 1, (2, 6, 32)), device="cuda", dtype=torch.float32)
    sb_cache_append(x, x, cache, ints([piece, (3, 0, 2, 6)]))
    with pytest.raises(ValueError, match="page index"):
        check_status()
    wc, ws = orc.append(x.double().cpu().numpy(), codes[0], scales[0], [(3, 0, 2, 6)])
    assert np.array_equal(cache.k.view(torch.uint8).cpu().numpy(), wc) and np.array_equal(cache.k_scale.cpu().numpy(), ws)


# ----------------------------------------------------------------------------------------------------------------- attention
class Problem:
    """Requests with given lengths and new tokens over a cache of normal keys and values; `lean` shifts the logits' mean by -lean."""

    def __init__(self, lengths, new, heads=2, kv=None, dim=64, page=16, dtype="bf16", lean=0.0, seed=0, halves=False, extra_rows=0, loud=1.0):
        from stickbreaking_attention_b200 import SbCache
        rng = np.random.default_rng(seed)
        kv = kv or heads
        self.lengths, self.new, self.heads, self.kv, self.dim, self.page, self.rng = list(lengths), list(new), heads, kv, dim, page, rng
        held = [-(-t // page) for t in lengths]
        pages, width = sum(held) + 3, max(held + [1]) + 1
        codes, scales, _ = filled_cache(rng, pages, kv, page, dim)
        for c in codes:
            c[rng.random(c.shape) < 0.02] = 127  # NaN in places that hold no token
        order = rng.permutation(pages)
        self.tables, at = np.full((len(lengths), width), -1), 0
        tilt = np.sqrt(lean / np.sqrt(dim))
        self.k, self.v = [], []  # [kv, L, dim] per request, as the cache holds them
        for r, t in enumerate(lengths):
            self.tables[r, :held[r]] = order[at:at + held[r]]
            at += held[r]
            kk, vv = np.zeros((2, kv, t, dim))
            for b in range(held[r]):
                n = min(page, t - b * page)
                for which, (c, s, out) in enumerate(zip(codes, scales, (kk, vv))):
                    x = rng.normal(0, loud, (kv, n, dim)) - (tilt if which == 0 else 0)
                    p = self.tables[r, b]
                    for g in range(kv):
                        s[p, g] = orc.scale_for(np.abs(x[g]).max())
                        c[p, g, :n, :dim] = orc.to_code(x[g] / s[p, g])
                        c[p, g, :n, dim:] = 0
                        out[g, b * page:b * page + n] = orc.VALUES[c[p, g, :n, :dim]] * s[p, g]
            self.k.append(kk)
            self.v.append(vv)
        self.codes, self.scales = codes, scales
        dev = lambda a, b: torch.tensor(np.stack([a, b], 1), device="cuda") if halves else [torch.tensor(x, device="cuda") for x in (a, b)]  # noqa: E731
        c, s = dev(*codes), dev(*scales)
        c, s = ([c[:, 0], c[:, 1]], [s[:, 0], s[:, 1]]) if halves else (c, s)
        self.cache = SbCache(*(x.view(torch.float8_e4m3fn) for x in c), *s)
        T = sum(new) + extra_rows
        self.q = torch.tensor(rng.normal(0, 1, (heads, T, dim)) + tilt, device="cuda").to(DTYPES[dtype])
        self.own_v = torch.tensor(rng.normal(0, 1, (kv, T, dim)), device="cuda").to(DTYPES[dtype])

    def widen(self):
        """Room for more pages in the tables, until the work that they allow is that of the kernel for many queries."""
        need = -(-2 ** 21 // (self.q.shape[0] * self.q.shape[1] * self.page))
        self.tables = np.pad(self.tables, ((0, 0), (0, max(0, need - self.tables.shape[1]))), constant_values=-1)
        return self

    def run(self, ends=True, **kw):
        from stickbreaking_attention_b200 import sb_attn_cached
        return sb_attn_cached(self.q, self.cache, ints(self.tables).reshape(len(self.lengths), -1), ints(self.lengths), ints(np.cumsum(self.new)) if ends else None, **kw)

    def want(self, inv_temp=None, attend_current=False, v=None, wide=False):
        """o, rem and their bounds without the rounding to the output's type."""
        inv_temp = self.dim ** -0.5 if inv_temp is None else inv_temp
        q = self.q.double().cpu().numpy()
        own = v.double().cpu().numpy() if v is not None else None
        terms = (2 if self.q.dtype == torch.float16 else 1) if wide else 0  # of bfloat16, for the weights
        outs, at = [[], [], [], []], 0
        for r, n in enumerate(self.new):
            rows = slice(at, at + n)
            at += n
            per = [orc.attend(q[h, rows], self.k[r][h * self.kv // self.heads], self.v[r][h * self.kv // self.heads], n, inv_temp, attend_current,
                              own[h * self.kv // self.heads, rows] if own is not None else None, terms) for h in range(self.heads)]
            for out, x in zip(outs, zip(*per)):
                out.append(np.stack(x))
        return [np.concatenate(x, 1) for x in outs]

    def check(self, ends=True, v=None, wide=False, **kw):
        o, rem = self.run(ends, v=v, **kw)
        rows = sum(self.new)
        assert o.shape == self.q.shape and rem.shape == self.q.shape[:2] and o.dtype == rem.dtype == self.q.dtype
        self.compare(o[:, :rows], rem[:, :rows], *self.want(v=v, wide=wide, **kw), own_v=v)
        assert (rem[:, rows:] == 0).all()
        return o, rem

    def compare(self, o, rem, wo, wr, to, tr, own_v=None):
        """The bounds, and half a step of the output's type (for subnormal results half the smallest one); with v, rem has been rounded before."""
        half, tiny = torch.finfo(o.dtype).eps / 2, torch.finfo(o.dtype).smallest_normal * torch.finfo(o.dtype).eps / 2
        go, gr = o.double().cpu().numpy(), rem.double().cpu().numpy()
        fr = tr + half * np.abs(wr) * (1 + half) + tiny
        fo = to + half * (np.abs(wo) + to) + tiny
        if own_v is not None:
            fo = fo + (half * wr + tiny)[..., None] * np.abs(np.repeat(own_v[:, :wo.shape[1]].double().cpu().numpy(), self.heads // self.kv, 0)) * (1 + 2 * half)
        assert np.isfinite(go).all() and np.isfinite(gr).all()
        assert (np.abs(gr - wr) <= fr).all(), float((np.abs(gr - wr) / fr).max())
        assert (np.abs(go - wo) <= fo).all(), float((np.abs(go - wo) / fo).max())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim, page", [(64, 16), (128, 64), (32, 32), (50, 16), (100, 128), (1, 16), (33, 64)])
@pytest.mark.parametrize("current", [False, True])
def test_single_tokens(dtype, dim, page, current):
    lengths = [1, 2, 15, 16, 17, 31, 33, 64, 65, 200, 391]
    p = Problem(lengths, [1] * len(lengths), heads=3, dim=dim, page=page, dtype=dtype, lean=3.0, seed=dim)
    p.check(ends=False, attend_current=current)


@pytest.mark.parametrize("shared", [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 33])
@pytest.mark.parametrize("dim", [64, 128])
def test_shared_heads(shared, dim):
    p = Problem([130, 1, 77], [1, 1, 1], heads=2 * shared, kv=2, dim=dim, page=32, dtype="bf16", lean=2.0, seed=shared)
    p.check(ends=False, v=p.own_v)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shared", [1, 3])
@pytest.mark.parametrize("current", [False, True])
@pytest.mark.parametrize("dim", [128, 40])
def test_several_new_tokens(dtype, shared, current, dim):
    lengths, new = [40, 1, 9, 100, 33, 300, 64, 5], [3, 1, 9, 17, 0, 70, 64, 2]
    p = Problem(lengths, new, heads=2 * shared, kv=2, dim=dim, page=16, dtype=dtype, lean=2.0, seed=1, extra_rows=5)
    p.check(attend_current=current)
    p.check(attend_current=current, v=p.own_v)


@pytest.mark.parametrize("dim, page", [(128, 64), (64, 16), (100, 32), (48, 128), (128, 16), (64, 64), (32, 64), (24, 16), (17, 128)])
@pytest.mark.parametrize("shared, lengths, new", [(1, [200], [100]), (4, [70, 1000, 300], [70, 100, 41]), (1, [700, 64, 129], [300, 64, 128]), (8, [333], [33]), (3, [2500], [90]), (1, [300, 150], [1, 60])])
@pytest.mark.parametrize("current", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_many_queries(dim, page, shared, lengths, new, current, dtype):
    """Tiles of 256 queries, full and not, one half of them empty, sequences of one step and of many, cut into shares."""
    p = Problem(lengths, new, heads=2 * shared, kv=2, dim=dim, page=page, dtype=dtype, lean=3.0, seed=dim + shared, extra_rows=3).widen()
    p.check(attend_current=current, v=p.own_v, wide=True)
    p.check(attend_current=current, wide=True)


def test_which_kernel_runs():
    """Few queries per key and little work take the one kernel, many queries of 16 bits the other."""
    from torch.profiler import ProfilerActivity, profile

    def kernels(p):
        p.run()
        with profile(activities=[ProfilerActivity.CUDA]) as prof:
            p.run()
            torch.cuda.synchronize()
        return " ".join(e.key for e in prof.key_averages())
    make = lambda dtype, new: Problem([300], [new], heads=8, kv=2, dim=64, page=16, dtype=dtype)  # noqa: E731
    names = kernels(make("bf16", 60))
    if "cached" not in names:
        pytest.skip("the profiler records no kernels here")
    assert "cached_tc_kernel" not in names
    assert "cached_tc_kernel" in kernels(make("bf16", 60).widen())
    assert "cached_tc_kernel" in kernels(make("f16", 60).widen())
    assert "cached_tc_kernel" not in kernels(make("f32", 60).widen())
    assert "cached_tc_kernel" not in kernels(make("bf16", 5).widen())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_many_queries_many_requests(dtype):
    rng = np.random.default_rng(1)
    lengths = [int(x) for x in rng.integers(0, 400, 90)]
    new = [min(t, int(n)) for t, n in zip(lengths, rng.integers(0, 260, 90))]
    Problem(lengths, new, heads=2, kv=1, dim=64, page=32, dtype=dtype, lean=2.0).widen().check(wide=True)


@pytest.mark.parametrize("case", ["far", "strong", "hot", "scaled"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_many_queries_extreme_logits(case, dtype):
    p = Problem([300, 150], [100, 90], heads=2, dim=64, page=16, dtype=dtype, lean=0.0, seed=3).widen()
    if case == "far":
        p.q = torch.full_like(p.q, -1.0)
        for r, t in enumerate(p.lengths):
            p.k[r][:] = 0.625
            for b in range(-(-t // 16)):
                p.cache.k.view(torch.uint8)[p.tables[r, b], :, :min(16, t - 16 * b)] = int(orc.to_code(np.float64(0.625)))
                p.cache.k_scale[p.tables[r, b]] = 1.0
    p.check(inv_temp={"far": 1.0, "strong": 4.0, "hot": 30.0, "scaled": 0.0}[case], wide=True)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_many_queries_strides(dtype):
    p = Problem([170, 133], [100, 60], heads=4, kv=2, dim=128, page=32, dtype=dtype, halves=True, lean=1.0).widen()
    flat = p.run(v=p.own_v)
    p.q = p.q.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    major = p.check(v=p.own_v.permute(1, 0, 2).contiguous().permute(1, 0, 2), wide=True)
    assert all(torch.equal(a, b) for a, b in zip(flat, major))
    odd = torch.zeros(4, p.q.shape[1], 131, device="cuda", dtype=p.q.dtype)
    odd[..., 1:129] = p.q
    p.q = odd[..., 1:129]  # rows that do not start at an aligned address
    assert all(torch.equal(a, b) for a, b in zip(flat, p.run(v=p.own_v)))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 32])
def test_many_queries_nan(dtype, dim):
    """NaN in a value that some queries of a tile see; in a key; in a value that all see."""
    p = Problem([350, 200], [100, 70], heads=2, dim=dim, page=16, dtype=dtype, lean=1.0).widen()
    clean_o, clean_rem = p.run()
    for key in (300, 20):  # rows 0 ... 99 are the tokens 250 ... 349
        page, place, sees = p.tables[0, key // 16], key % 16, max(0, key + 1 - 250)
        codes = p.cache.v.view(torch.uint8)
        was = int(codes[page, 1, place, 9])
        codes[page, 1, place, 9] = 255
        o, rem = p.run()
        bad = torch.zeros_like(o, dtype=torch.bool)
        bad[1, sees:100, 9] = True
        assert o[bad].isnan().all() and torch.equal(o[~bad], clean_o[~bad]) and torch.equal(rem, clean_rem)
        codes[page, 1, place, 9] = was
    page, place = p.tables[0, 300 // 16], 300 % 16
    p.cache.k.view(torch.uint8)[page, 0, place, 3] = 127
    o, rem = p.run()
    bad = torch.zeros_like(o, dtype=torch.bool)
    bad[0, 51:100] = True
    assert o[bad].isnan().all() and not o[~bad].isnan().any() and rem[0, 51:100].isnan().all() and int(rem.isnan().sum()) == 49


@pytest.mark.parametrize("what", ["largest", "smallest", "far scales", "infinite"])
def test_many_queries_float16_range(what):
    """Queries at both ends of float16; pages of values whose scales lie 2^60 apart; an infinite query."""
    p = Problem([300, 150], [100, 90], heads=2, dim=64, page=16, dtype="f16", lean=1.0, seed=4).widen()
    if what == "far scales":  # results are in float16: the small pages' share of them is lost, the large ones' must not suffer
        for r, t in enumerate(p.lengths):
            for b in range(0, -(-t // 16), 2):
                p.cache.v_scale[p.tables[r, b]] *= 2.0 ** -60
                p.v[r][:, 16 * b:16 * b + 16] *= 2.0 ** -60
        p.check(wide=True)
        return
    if what == "infinite":
        clean = p.run()
        p.q[1, 7, 3] = torch.inf
        o, rem = p.run()
        rest = torch.ones_like(rem, dtype=torch.bool)
        rest[1, 7] = False
        assert torch.equal(o[rest], clean[0][rest]) and torch.equal(rem[rest], clean[1][rest])
        return
    p.q = p.q * (2.0 ** 13 if what == "largest" else 2.0 ** -22)
    assert p.q.isfinite().all() and p.q.abs().max() > 2 ** 14 if what == "largest" else (p.q.abs() < 2.0 ** -14).all()
    p.check(inv_temp=2.0 ** -16 if what == "largest" else 2.0 ** 19, wide=True)


@pytest.mark.parametrize("page_index", [-1, 10 ** 6])
def test_many_queries_bad_pages(page_index, monkeypatch):
    from stickbreaking_attention_b200 import check_status
    monkeypatch.setenv("SBATTN_CHECK_STATUS", "0")
    p = Problem([350, 200], [100, 70], heads=2, dim=64, page=16, dtype="bf16").widen()
    good = p.run()
    p.tables[0, 3] = page_index
    o, rem = p.run()
    with pytest.raises(ValueError, match="page index"):
        check_status()
    assert torch.equal(o[:, 100:], good[0][:, 100:]) and torch.equal(rem[:, 100:], good[1][:, 100:])


@pytest.mark.parametrize("lean", [0.0, 3.0, 8.0])
def test_long(lean):
    p = Problem([5000, 3, 2049], [1, 1, 1], heads=2, dim=64, page=64, dtype="f32", lean=lean, seed=7)
    p.check(ends=False)


def test_many_requests():
    rng = np.random.default_rng(1)
    lengths = [int(x) for x in rng.integers(0, 90, 700)]
    new = [min(t, int(n)) for t, n in zip(lengths, rng.integers(0, 4, 700))]
    Problem(lengths, new, heads=1, dim=32, page=16, dtype="f32", lean=2.0).check()


def test_most_requests():
    """2048 requests; one more is refused."""
    from stickbreaking_attention_b200 import sb_attn_cached
    rng = np.random.default_rng(1)
    lengths = [int(x) for x in rng.integers(0, 20, 2048)]
    new = [min(t, int(n)) for t, n in zip(lengths, rng.integers(0, 3, 2048))]
    p = Problem(lengths, new, heads=1, dim=16, page=16, dtype="f32", lean=2.0)
    p.check()
    with pytest.raises(ValueError, match="2048 requests"):
        sb_attn_cached(p.q, p.cache, ints(np.zeros((2049, 1))), ints(np.zeros(2049)), ints(np.zeros(2049)))


@pytest.mark.parametrize("wide", [False, True])
def test_long_caches(wide):
    """Pages behind the first 4 GB of codes and their scales: read, and written by an append."""
    from stickbreaking_attention_b200 import SbCache, sb_cache_append
    p = Problem([300, 200], [90, 70] if wide else [1, 3], heads=8, kv=8, dim=128, page=64, dtype="bf16", lean=3.0)
    if wide:
        p.widen()
    small, base = p.cache, 70000  # 64 KB a page
    n = small.k.shape[0]
    big = [torch.empty(base + n, *x.shape[1:], dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for x in small[:2]]
    big += [torch.empty(base + n, 8, dtype=torch.float32, device="cuda") for _ in range(2)]
    for b, x in zip(big, small):
        (b.view(torch.uint8) if b.dtype != torch.float32 else b)[base:] = x.view(torch.uint8) if b.dtype != torch.float32 else x
    p.cache = SbCache(*big)
    flat = p.tables.copy()
    p.tables = np.where(flat >= 0, flat + base, flat)
    p.check(wide=wide)
    x = torch.randn(8, 5, 128, device="cuda", dtype=torch.bfloat16)
    page = int(p.tables[0, 0])
    sb_cache_append(x, x, p.cache, ints([(page, 0, 3, 5)]))
    wc, ws = orc.append(x.double().cpu().numpy(), p.codes[0][flat[0, 0]][None], p.scales[0][flat[0, 0]][None], [(0, 0, 3, 5)])
    assert np.array_equal(p.cache.k[page].view(torch.uint8).cpu().numpy(), wc[0]) and np.array_equal(p.cache.k_scale[page].cpu().numpy(), ws[0].astype(np.float32))


def test_strides_and_halves():
    p = Problem([70, 33], [4, 1], heads=4, kv=2, dim=64, page=16, dtype="bf16", halves=True, lean=1.0)
    flat = p.run(v=p.own_v)
    p.q = p.q.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    major = p.check(v=p.own_v.permute(1, 0, 2).contiguous().permute(1, 0, 2))
    assert all(torch.equal(a, b) for a, b in zip(flat, major))
    p.q = torch.stack([p.q, p.q], -1)[..., 0]
    assert all(torch.equal(a, b) for a, b in zip(flat, p.run(v=torch.stack([p.own_v] * 2, -1)[..., 0])))
    p.q = p.q[:1].expand(4, -1, -1)  # one head for all
    p.check()


def test_empty_requests_and_rows():
    """Requests of length 0, without rows, without keys to see; rows behind the last end."""
    from stickbreaking_attention_b200 import sb_attn_cached
    p = Problem([0, 20, 0, 1], [0, 1, 0, 1], dim=32, dtype="f32", extra_rows=3)
    o, rem = p.check()
    assert (rem[:, 1] == 1).all() and (o[:, 1] == 0).all()  # the first token of a request sees nothing
    q = torch.randn(2, 6, 32, device="cuda")  # without ends: a row per request, those of empty requests not covered, two rows more
    o, rem = sb_attn_cached(q, p.cache, ints(p.tables), ints(p.lengths))
    assert (rem[:, [0, 2, 4, 5]] == 0).all() and (rem[:, 3] == 1).all() and (o[:, 3] == 0).all() and (rem[:, 1] > 0).all()
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    o, rem = sb_attn_cached(q, p.cache, none.view(0, 2), none, none)
    assert (rem == 0).all()
    o, rem = sb_attn_cached(q[:, :0], p.cache, none.view(0, 2), none, none)
    assert o.shape == (2, 0, 32)


@pytest.mark.parametrize("case", ["far", "strong", "dead", "hot", "scaled"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_extreme_logits(case, dtype):
    """Weights near 2^-60 everywhere, sticks that one key takes, values of scales 2^40 apart behind a stick that is used up."""
    p = Problem([150, 64, 7], [2, 1, 1], heads=2, dim=64, page=16, dtype=dtype, lean=0.0, seed=3)
    temp = {"far": 1.0, "strong": 4.0, "dead": 1.0, "hot": 30.0, "scaled": 0.0}[case]
    if case in ("far", "dead"):
        p.q = torch.full_like(p.q, -1.0 if case == "far" else 1.0)
        for r, t in enumerate(p.lengths):
            p.k[r][:] = 0.625
            for b in range(-(-t // 16)):
                n, page = min(16, t - 16 * b), p.tables[r, b]
                p.cache.k.view(torch.uint8)[page, :, :n] = int(orc.to_code(np.float64(0.625)))
                p.cache.k_scale[page] = 1.0
                if case == "dead":
                    s = 2.0 ** (20 if b == 0 else -20)
                    p.v[r][:, 16 * b:16 * b + n] *= (s / p.scales[1][page])[:, None, None]
                    p.cache.v_scale[page] = s
    p.check(inv_temp=temp)


def test_nan_stays_with_those_who_see_it():
    """NaN in a key or value: results of the tokens and heads that see it are NaN (in a value: in its column), no others."""
    p = Problem([50, 40], [6, 1], heads=2, dim=64, page=16, dtype="f32", lean=1.0)
    clean_o, clean_rem = p.run()
    page, place = p.tables[0, 47 // 16], 47 % 16  # key 47 of request 0: its rows are the tokens 44 ... 49
    p.cache.v.view(torch.uint8)[page, 1, place, 9] = 127
    o, rem = p.run()
    bad = torch.zeros_like(o, dtype=torch.bool)
    bad[1, 4:6, 9] = True
    assert o[bad].isnan().all() and torch.equal(o[~bad], clean_o[~bad]) and torch.equal(rem, clean_rem)
    p.cache.v.view(torch.uint8)[page, 1, place, 9] = 255
    o, rem = p.run(attend_current=True)
    assert o[1, 3:6, 9].isnan().all() and int(o.isnan().sum()) == 3
    p.cache.v.view(torch.uint8)[page, 1, place, 9] = 0
    p.cache.k.view(torch.uint8)[page, 0, place, 3] = 127
    o, rem = p.run()
    bad = torch.zeros_like(o, dtype=torch.bool)
    bad[0, 4:6] = True
    assert o[bad].isnan().all() and not o[~bad].isnan().any() and rem[0, 4:6].isnan().all() and int(rem.isnan().sum()) == 2
    p.q[1, 2, 5] = float("inf")
    o, rem = p.run()
    assert not o[1, :2].isnan().any() and not o[1, 3:].isnan().any()


@pytest.mark.parametrize("page_index", [-1, 10 ** 6, 2147483647, -2147483648])
def test_bad_pages_are_reported(page_index, monkeypatch):
    from stickbreaking_attention_b200 import check_status
    monkeypatch.setenv("SBATTN_CHECK_STATUS", "0")
    p = Problem([50, 40], [2, 1], heads=2, dim=64, page=16, dtype="bf16")
    good = p.run()
    p.tables[0, 1] = page_index
    o, rem = p.run()
    with pytest.raises(ValueError, match="page index"):
        check_status()
    assert torch.equal(o[:, 2:], good[0][:, 2:]) and torch.equal(rem[:, 2:], good[1][:, 2:])  # the other request is not touched by it


@pytest.mark.parametrize("what", ["short", "long", "negative", "order", "beyond"])
def test_bad_lengths_are_reported(what, monkeypatch):
    from stickbreaking_attention_b200 import check_status, sb_attn_cached
    monkeypatch.setenv("SBATTN_CHECK_STATUS", "0")
    p = Problem([50, 40, 30], [2, 1, 2], heads=2, dim=64, page=16, dtype="bf16")
    lengths, ends = {"short": ([1, 40, 30], [2, 3, 5]), "long": ([5000, 40, 30], [2, 3, 5]), "negative": ([-4, 40, 30], [2, 3, 5]),
                     "order": ([50, 40, 30], [4, 3, 5]), "beyond": ([50, 40, 30], [2, 3, 9])}[what]
    sb_attn_cached(p.q, p.cache, ints(p.tables), ints(lengths), ints(ends))
    with pytest.raises(ValueError, match="rejected"):
        check_status()


def test_refusals():
    from stickbreaking_attention_b200 import SbCache, sb_attn_cached, sb_cache_append, sb_cache_blocks
    p = Problem([50, 40], [1, 1], heads=4, kv=2, dim=64, page=16, dtype="bf16")
    c, t, n, pieces = p.cache, ints(p.tables), ints(p.lengths), ints([(0, 0, 0, 1)])
    q = p.q

    def attend(error, q=q, c=c, t=t, n=n, **kw):
        with pytest.raises(error):
            sb_attn_cached(q, c, t, n, **kw)
    attend(ValueError, q=q[:3])
    attend(ValueError, q=q[0])
    attend(TypeError, q=q.double())
    attend(ValueError, q=torch.randn(4, 2, 32, device="cuda"))
    attend(ValueError, q=torch.randn(4, 2, 129, device="cuda"))
    attend(ValueError, q=q[:, :1])
    attend(TypeError, n=n.long())
    attend(TypeError, t=t.long())
    attend(ValueError, t=t[:1])
    attend(ValueError, n=n.cpu())
    attend(ValueError, ends=n[:1])
    attend(TypeError, ends=n.long())
    attend(TypeError, v=p.own_v.float())
    attend(ValueError, v=p.own_v[:1])
    attend(TypeError, c=c._replace(k=c.k.view(torch.uint8)))
    attend(TypeError, c=c._replace(k_scale=c.k_scale.half()))
    attend(ValueError, c=c._replace(v=c.v[:1]))
    attend(ValueError, c=c._replace(v_scale=c.v_scale[:1]))
    attend(ValueError, c=SbCache(*(x[:0] for x in c)))
    attend(ValueError, c=c._replace(k=c.k[:, :, :, ::2], v=c.v[:, :, :, ::2]))
    attend(ValueError, c=c._replace(k=c.k.transpose(0, 1).contiguous().transpose(0, 1)))
    attend(RuntimeError, q=q.clone().requires_grad_())
    attend(RuntimeError, v=p.own_v.clone().requires_grad_())
    attend(ValueError, c=c._replace(k=c.k.cpu()))
    with torch.no_grad():
        sb_attn_cached(q.clone().requires_grad_(), c, t, n)
    for k, v, pc in ((p.own_v, p.own_v[:, :1], pieces), (q, q, pieces), (p.own_v, p.own_v.float(), pieces), (p.own_v, p.own_v, pieces.long()), (p.own_v, p.own_v, pieces[:, :3])):
        with pytest.raises((ValueError, TypeError)):
            sb_cache_append(k, v, c, pc)
    for k, v in ((p.own_v.clone().requires_grad_(), p.own_v), (p.own_v, p.own_v.clone().requires_grad_())):  # the cache would lose the gradient
        with pytest.raises(RuntimeError, match="backward"):
            sb_cache_append(k, v, c, ints([(-1, 0, 0, 0)]))
        with torch.no_grad():
            sb_cache_append(k, v, c, ints([(-1, 0, 0, 0)]))
    free, count = ints([0, 1]), ints([2])
    for bad in (dict(page_tokens=20), dict(lengths=n.long()), dict(new_tokens=n[:1]), dict(tables=t[:1]), dict(tokens=-1), dict(free_count=ints([1, 2])), dict(free_pages=free.cpu()),
                dict(tables=t[:, ::2]), dict(free_pages=ints([0, 1, 2, 3])[::2]), dict(tables=t[:1].expand(2, -1))):
        with pytest.raises((ValueError, TypeError)):
            sb_cache_blocks(**{**dict(lengths=n, new_tokens=ints([1, 1]), tables=t, free_pages=free, free_count=count, page_tokens=16, tokens=2), **bad})


# ------------------------------------------------------------------------------------------------------------------ together
def serve(graph, dtype=torch.bfloat16, steps=6, stream=None):
    """Prompts, then single tokens, through the three operators, as a program serves them; returns results, and the inputs."""
    from stickbreaking_attention_b200 import sb_attn_cached, sb_cache, sb_cache_append, sb_cache_blocks
    g = torch.Generator(device="cuda").manual_seed(0)
    R, H, kv, D, P, T0 = 4, 4, 2, 64, 16, 60
    cache = sb_cache(40, kv, D, P)
    lengths, tables, free, count = ints([0] * R), torch.full((R, 12), -1, dtype=torch.int32, device="cuda"), ints(np.arange(40)[::-1]), ints([40])
    new_prompt = ints([20, 1, 33, 0])
    randn = lambda h, t: torch.randn(h, t, D, generator=g, device="cuda").to(dtype)  # noqa: E731

    def step(q, k, v, new, tokens):
        s = sb_cache_blocks(lengths, new, tables, free, count, P, tokens)
        sb_cache_append(k, v, cache, s.pieces)
        out = sb_attn_cached(q, cache, tables, s.lengths, s.ends, v=v)
        lengths.copy_(s.lengths)
        count.copy_(s.free_count)
        return out
    seen = [(randn(H, T0), randn(kv, T0), randn(kv, T0), new_prompt.tolist())]
    outs = [step(*seen[0][:3], new_prompt, T0)]
    bufs = [torch.zeros(h, R, D, device="cuda", dtype=dtype) for h in (H, kv, kv)]
    new = ints([0] * R)
    runner = None
    if graph:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*bufs, new, R)  # takes no tokens: changes nothing
        torch.cuda.current_stream().wait_stream(side)
        runner = torch.cuda.CUDAGraph()
        with torch.cuda.graph(runner):
            static = step(*bufs, new, R)
    for i in range(steps):
        many = [1, 1, 1, 1] if i != 3 else [1, 0, -33 - 3, 1]  # in step 3 one request waits and one ends
        new.copy_(ints(many))
        data = [randn(h, R) for h in (H, kv, kv)]
        for b, d in zip(bufs, data):
            b.copy_(d)
        if runner:
            runner.replay()
            outs.append(tuple(x.clone() for x in static))
        else:
            outs.append(step(*bufs, new, R))
        seen.append((*data, many))
    torch.cuda.synchronize()
    return outs, seen, cache, tables, lengths, count


def test_serving_run(monkeypatch):
    monkeypatch.setenv("SBATTN_CHECK_STATUS", "0")
    from stickbreaking_attention_b200 import check_status
    outs, seen, cache, tables, lengths, count = serve(False)
    captured = serve(True)
    check_status()
    # every step against the oracle, over the keys and values as the cache rounds them
    page, kv, D, H = 16, 2, 64, 4
    model = np.zeros((40, kv, page, 64), np.uint8), np.zeros((40, kv)), np.zeros((40, kv, page, 64), np.uint8), np.zeros((40, kv))
    state = np.zeros(4, int), np.full((4, 12), -1), np.arange(40)[::-1].copy(), 40
    for (o, rem), (q, k, v, new), (co, crem) in zip(outs, seen, captured[0]):
        T = q.shape[1]
        after, cnt, ends, _, pieces, tab, free = orc.blocks(state[0], np.array(new), state[1], state[2], state[3], page, T)
        state = after, tab, free, cnt
        kc, ks = orc.append(k.double().cpu().numpy(), model[0], model[1], pieces)
        vc, vs = orc.append(v.double().cpu().numpy(), model[2], model[3], pieces)
        model = kc, ks, vc, vs
        p = Problem.__new__(Problem)
        p.heads, p.kv, p.dim, p.q = H, kv, D, q
        p.lengths, p.new = list(after), [max(0, n) for n in new]
        held = [tab[r, :-(-t // page)] for r, t in enumerate(after)]
        deq = lambda c, s, x, t: (orc.VALUES[c[x]] * s[x][..., None, None]).transpose(1, 0, 2, 3).reshape(kv, -1, 64)[:, :t]  # noqa: E731
        p.k = [deq(kc, ks, x, t) for x, t in zip(held, after)]
        p.v = [deq(vc, vs, x, t) for x, t in zip(held, after)]
        rows = sum(p.new)
        p.compare(o[:, :rows], rem[:, :rows], *p.want(v=v), own_v=v)
        assert (rem[:, rows:] == 0).all()
        assert torch.equal(o[:, :rows], co[:, :rows]) and torch.equal(rem, crem)
    assert np.array_equal(cache.k.view(torch.uint8).cpu().numpy(), model[0]) and np.array_equal(cache.v_scale.cpu().numpy(), model[3])
    assert lengths.tolist() == list(state[0]) and count.tolist() == [state[3]]
    for a, b in ((cache.k.view(torch.uint8), captured[2].k.view(torch.uint8)), (tables, captured[3]), (lengths, captured[4]), (count, captured[5])):
        assert torch.equal(a, b)


def test_same_answer_as_whole_sequences():
    """Token by token over the cache against sb_attn_varlen over the rounded keys and values: both are within their own roundings of the definition."""
    from stickbreaking_attention_b200 import sb_attn_varlen
    p = Problem([97, 300], [97, 300], heads=2, dim=64, page=32, dtype="f32", lean=2.0)
    k, v = (torch.tensor(np.concatenate(x, 1), device="cuda", dtype=torch.float32) for x in (p.k, p.v))
    o, rem = p.check()
    wo, wrem = sb_attn_varlen(p.q, k, v, ints([97, 397]), 300, zero_start=False)
    assert (o - wo).abs().max() < 2e-5 and (rem - wrem).abs().max() < 2e-5


def test_other_streams_and_repeats():
    p = Problem([2000, 77, 640], [1, 1, 1], heads=4, kv=2, dim=128, page=64, dtype="bf16", lean=5.0)
    first = p.run(ends=False)
    outs = []
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for i in range(12):  # calls that overlap, on several streams
        with torch.cuda.stream(streams[i % 3]):
            outs.append(p.run(ends=False))
    torch.cuda.synchronize()
    for o, rem in outs:
        assert torch.equal(o, first[0]) and torch.equal(rem, first[1])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_many_queries_on_several_streams(dtype):
    p = Problem([700, 77, 640], [300, 40, 70], heads=4, kv=2, dim=64, page=64, dtype=dtype, lean=5.0).widen()
    first = p.run(v=p.own_v)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(p.run(v=p.own_v))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for out in outs for a, b in zip(out, first))


@pytest.mark.parametrize("wide", [False, True])
def test_broadcast_inputs(wide):
    """One query for all heads and one value for all tokens, as views of stride 0; one row of page indexes for all requests."""
    from stickbreaking_attention_b200 import sb_attn_cached, sb_cache_append
    p = Problem([170, 170], [70, 60] if wide else [2, 1], heads=4, kv=2, dim=64, page=16, dtype="bf16", lean=1.0)
    if wide:
        p.widen()
    T = p.q.shape[1]
    q, v = p.q[:1].expand(4, -1, -1), p.own_v[:, :1].expand(-1, T, -1)
    t = ints(p.tables[:1]).expand(2, -1)
    n, ends = ints(p.lengths), ints(np.cumsum(p.new))
    a, b = sb_attn_cached(q, p.cache, t, n, ends, v=v), sb_attn_cached(q.contiguous(), p.cache, t.contiguous(), n, ends, v=v.contiguous())
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and a[0].is_contiguous()
    piece = ints([(int(p.tables[0, 3]), 0, 0, min(T, 16))])
    sb_cache_append(v, v, p.cache, piece)
    one = [x.view(torch.uint8).clone() for x in p.cache[:2]]
    sb_cache_append(v.contiguous(), v.contiguous(), p.cache, piece)
    assert all(torch.equal(x, y.view(torch.uint8)) for x, y in zip(one, p.cache[:2]))


def test_results_do_not_depend_on_the_neighbours_values():
    """The same request beside others of the same lengths but other contents gives the same bits."""
    a = Problem([300, 500], [1, 3], heads=2, dim=64, page=16, dtype="bf16", lean=3.0, seed=1)
    o, rem = a.run()
    other = a.tables[0]
    for page in other[other >= 0]:
        a.cache.k.view(torch.uint8)[page] = 127
        a.cache.v.view(torch.uint8)[page] = 127
    o2, rem2 = a.run()
    assert torch.equal(o[:, 1:], o2[:, 1:]) and torch.equal(rem[:, 1:], rem2[:, 1:])


def test_torch_compile():
    """A step inside torch.compile(fullgraph=True): the same bits, tables and cache included."""
    from stickbreaking_attention_b200 import sb_attn_cached, sb_cache, sb_cache_append, sb_cache_blocks

    def step(q, k, v, cache, lengths, new, tables, free, count):
        s = sb_cache_blocks(lengths, new, tables, free, count, 16, 9)
        sb_cache_append(k, v, cache, s.pieces)
        o, rem = sb_attn_cached(q, cache, tables, s.lengths, s.ends, v=v)
        return o * 2, rem, s.lengths, s.free_count, s.slots

    outs = []
    for run in (step, torch.compile(step, backend="aot_eager", fullgraph=True)):
        g = torch.Generator(device="cuda").manual_seed(1)
        cache, tables = sb_cache(12, 2, 64, 16), torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
        lengths, free, count = ints([0, 0, 0]), ints(np.arange(12)), ints([12])
        for new in ([4, 0, 5], [1, 7, 1]):
            q, k, v = (torch.randn(9, h, 64, generator=g, device="cuda").bfloat16().transpose(0, 1) for h in (4, 2, 2))
            res = run(q, k, v, cache, lengths, ints(new), tables, free, count)
            lengths, count = res[2], res[3]
            outs.append((*(x.clone() for x in res), cache.k.view(torch.uint8).clone(), cache.v_scale.clone(), tables.clone(), free.clone()))
    for a, b in zip(outs[:2], outs[2:]):
        assert a[0].stride() == b[0].stride()
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_two_captured_graphs_and_an_eager_call(monkeypatch):
    """Graphs captured one after the other (their workspaces may come from one pool) and replayed in turn, with eager calls between."""
    monkeypatch.setenv("SBATTN_CHECK_STATUS", "0")
    ps = [Problem([300, 77], [1, 1], heads=4, kv=2, dim=128, page=64, dtype="bf16", lean=3.0, seed=1), Problem([900, 200], [70, 65], heads=4, kv=2, dim=64, page=16, dtype="bf16", lean=3.0, seed=2).widen()]
    from stickbreaking_attention_b200 import sb_attn_cached
    args = [(p.q, p.cache, ints(p.tables), ints(p.lengths), ints(np.cumsum(p.new))) for p in ps]
    want = [p.run() for p in ps]
    pool, graphs, outs = torch.cuda.graph_pool_handle(), [], []
    for a in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append([sb_attn_cached(*a) for _ in range(2)][1])
        graphs.append(g)
    for i in (0, 1, 1, 0, 1):
        graphs[i].replay()
        eager = ps[1 - i].run()
        assert torch.equal(outs[i][0], want[i][0]) and torch.equal(outs[i][1], want[i][1])
        assert torch.equal(eager[0], want[1 - i][0]) and torch.equal(eager[1], want[1 - i][1])


def test_torch_compile_refuses_gradients():
    from stickbreaking_attention_b200 import sb_attn_cached, sb_cache_append
    p = Problem([50], [1], heads=2, dim=64, page=16, dtype="bf16")
    x, piece = p.own_v.clone().requires_grad_(), ints([(-1, 0, 0, 0)])
    with pytest.raises(Exception, match="no backward"):
        torch.compile(lambda x: sb_cache_append(x, x, p.cache, piece))(x)
    with pytest.raises(Exception, match="backward"):
        torch.compile(lambda x: sb_attn_cached(x, p.cache, ints(p.tables), ints(p.lengths))[0].float().sum())(x).backward()
