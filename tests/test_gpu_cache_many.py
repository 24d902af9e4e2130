"""Attention over the 8-bit paged cache, many queries per key: blocks that go from tile to tile of different widths."""
import numpy as np
import pytest
import torch

from oracle import cache_oracle as orc
from test_gpu_cache import Problem

pytestmark = pytest.mark.gpu


class Rows(Problem):
    """A Problem whose oracle works on all rows of a request and head at once."""

    def want(self, inv_temp=None, attend_current=False, v=None, wide=False):
        inv_temp = self.dim ** -0.5 if inv_temp is None else inv_temp
        q = self.q.double().cpu().numpy()
        own = v.double().cpu().numpy() if v is not None else None
        terms = 2 if wide else 0  # of bfloat16, for the weights
        shared, outs, at = self.heads // self.kv, [[], [], [], []], 0
        for r, n in enumerate(self.new):
            rows = slice(at, at + n)
            at += n
            per = [orc.attend_rows(q[h, rows], self.k[r][h // shared], self.v[r][h // shared], n, inv_temp, attend_current, own[h // shared, rows] if own is not None else None, terms)
                   for h in range(self.heads)]
            for out, x in zip(outs, zip(*per)):
                out.append(np.stack(x))
        return [np.concatenate(x, 1) for x in outs]

    def other_powers(self):
        """Queries whose largest values lie in different powers of two from request to request, at the same logits."""
        at = 0
        for r, n in enumerate(self.new):
            e = r * 5 % 13 - 6
            self.q[:, at:at + n] *= 2.0 ** e
            self.k[r] *= 2.0 ** -e
            pages = self.tables[r][self.tables[r] >= 0]
            self.cache.k_scale[torch.tensor(pages, device="cuda")] *= 2.0 ** -e
            at += n
        return self


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim, page", [(128, 64), (64, 16), (32, 32)])
def test_narrow_tiles_before_full_ones(dim, page, dtype):
    """Tiles of at most 128 columns, whose second half of rows has nothing to do, one behind the other before a tile that has work for it: 2 to 5 and more of them, the full tile
    at every number of jobs modulo four (tiles' queries have two places in turn, their marks four).  Logits are of order one; factors of
    queries differ from request to request, so that those of another tile give other results."""
    rng = np.random.default_rng(dim)
    count = 13 * sms() // 8  # about thirteen tiles a block
    lengths = [int(x) for x in rng.integers(64, 129, count)]
    lengths[::9] = [x + 200 for x in lengths[::9]]
    new = [int(rng.integers(1, 33)) if r % 2 else 64 for r in range(count)]  # 4 ... 128 columns, or 256
    p = Rows(lengths, new, heads=32, kv=8, dim=dim, page=page, dtype=dtype, lean=2.0, seed=dim).other_powers()
    runs, places = set(), set()
    for tiles in orc.tiles_of_blocks(lengths, new, 8, 4, sms()):
        run = 0
        for i, (cols, steps) in enumerate(t for t in tiles if t[1] > 0):
            if cols > 128 and run > 1:
                runs.add(run)
                places.add(i % 4)
            run = run + 1 if cols <= 128 else 0
    assert {2, 3, 4, 5} <= runs and places == {0, 1, 2, 3}
    p.check(v=p.own_v, wide=True)


@pytest.mark.parametrize("lengths, new", [([1000] * 64, [20, 200] * 32), ([2000] * 64, [1] * 7 + [512])])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_single_tokens_beside_prompt_pieces(lengths, new, dtype):
    """A step of a server: some requests bring one token or a few, others the next piece of a prompt.  Against the same requests one kind at a time, which
    no tile of the other kind stands beside: the same weights in other shares, which changes float32 sums and the rounding of a few results."""
    from stickbreaking_attention_b200 import sb_attn_cached, SbCache
    new = (new * 64)[:64]
    kv, dim, page, T = 8, 128, 64, sum(new)
    g = torch.Generator(device="cuda").manual_seed(5)
    held = -(-lengths[0] // page)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    codes = [normal(64 * held, kv, page, dim).mul_(60).clamp_(-448, 448).to(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.full((64 * held, kv), 2.0 ** -6, device="cuda") for _ in range(2)]
    cache = SbCache(*codes, *scales)
    tables = torch.randperm(64 * held, generator=g, device="cuda").int().view(64, held)
    q = normal(4 * kv, T, dim).to(torch.bfloat16 if dtype == "bf16" else torch.float16)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    ends = np.cumsum(new)
    o, rem = sb_attn_cached(q, cache, tables, n, torch.tensor(ends, dtype=torch.int32, device="cuda"))
    for kind in sorted(set(new)):
        pick = [r for r in range(64) if new[r] == kind]
        rows = torch.cat([torch.arange(ends[r] - new[r], ends[r]) for r in pick]).cuda()
        at = torch.tensor(pick, device="cuda")
        mine = torch.tensor(np.cumsum([kind] * len(pick)), dtype=torch.int32, device="cuda")
        wo, wrem = sb_attn_cached(q[:, rows], cache, tables[at], n[at], mine)
        # two results of one number, each rounded to the type; on either side weights may have been rounded to a bfloat16 term, 2^-8 of the sum of
        # |weight * value|, which is at most the largest |value|; eight roundings of 2^-24 a key for the products of 1 - beta
        top = 448 * 2.0 ** -6
        half = torch.finfo(q.dtype).eps / 2
        assert ((o[:, rows].double() - wo.double()).abs() <= 2 * half * wo.double().abs() * (1 + half) + 2 * top * (2.0 ** -8 + 2000 * 8 * 2.0 ** -24)).all()
        assert ((rem[:, rows].double() - wrem.double()).abs() <= 2 * half * wrem.double() * (1 + half) + 2 * (2000 * 8 * 2.0 ** -24 * wrem.double() + 2.0 ** -29)).all()


# ------------------------------------------------------------------------------------------------------ weights
def built(logits, length, new, value_at, dtype, dim=64, page=16):
    """One request whose keys have the given logits (e4m3 values; -16 elsewhere) for every query, and a value of one at `value_at`, zero elsewhere."""
    p = Rows([length], [new], heads=2, kv=1, dim=dim, page=page, dtype=dtype).widen()
    x = np.full(length, -16.0)
    for key, t in logits.items():
        x[key] = t
    p.k, p.v = [np.zeros((1, length, dim))], [np.zeros((1, length, dim))]
    p.k[0][0, :, 0] = x
    p.v[0][0, value_at, 0] = p.v[0][0, value_at, 1] = 1.0
    for codes, scales, y in ((p.cache.k, p.cache.k_scale, p.k[0]), (p.cache.v, p.cache.v_scale, p.v[0])):
        scales.fill_(1.0)
        for b in range(-(-length // page)):
            n = min(page, length - b * page)
            codes.view(torch.uint8)[int(p.tables[0, b]), 0, :n] = torch.tensor(orc.to_code(y[0, b * page:b * page + n]), device="cuda")
    p.q.zero_()
    p.q[..., 0] = 1.0
    return p


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("first", [36, 40, 44, 48, 260, 264, 268, 272])
@pytest.mark.parametrize("logit", [5.0, 6.0, 10.0, 14.0, 18.0])
def test_strong_keys_behind_a_stick_that_is_partly_used(first, logit, dtype):
    """Four neighbouring keys whose logits pass the clamp of 1 - beta, with a key to their right that leaves 2^-7 to 2^-26 of the stick: the rightmost of the four takes
    all of that, and nothing of it may be lost to products of 1 + e that leave float32's range.  In steps that all queries see, and in the one that some do."""
    built({**{first + i: 24.0 for i in range(4)}, first + 5: logit}, 300, 40, first + 3, dtype).check(inv_temp=1.0, wide=True)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_strong_keys_one_behind_the_other(dtype):
    """Strong and middling keys at every place of a group: each takes its part of what the ones to its right have left."""
    for shift in range(4):
        logits = {100 + shift + i: t for i, t in enumerate([22.0, 4.0, 24.0, 1.0, 3.5, 20.0, 2.0, 0.5, 6.0, 5.0, 3.0])}
        for at in (100 + shift, 103 + shift, 105 + shift, 108 + shift):
            built(logits, 300, 40, at, dtype).check(inv_temp=1.0, wide=True)


@pytest.mark.parametrize("dim, page", [(128, 64), (64, 16), (32, 32)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_weights_keep_sixteen_bits(dim, page, dtype):
    """A prompt piece gets the weights that single tokens get but for 2^-16 of them, whatever type its queries have: what is left is the rounding of the results."""
    p = Rows([300, 700, 150], [64, 200, 90], heads=8, kv=2, dim=dim, page=page, dtype=dtype, lean=3.0, seed=dim).widen()
    p.check(wide=True)
    p.check(attend_current=True, v=p.own_v, wide=True)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("queries", [-129, -118, -60, 60, 105])
def test_bfloat16_range(queries, wide):
    """Queries at both ends of bfloat16, subnormal ones among them, and keys whose scales bring the logits back to order one."""
    p = Rows([300, 150], [100, 90] if wide else [3, 1], heads=4, kv=2, dim=64, page=16, dtype="bf16", lean=1.0, seed=6)
    if wide:
        p.widen()
    keys = min(-queries, 124)  # the largest scale is 2^118: 448 times it is still a float32 number
    p.q = (p.q.double() * 2.0 ** queries).to(torch.bfloat16)
    for r in range(2):
        p.k[r] *= 2.0 ** keys
    p.cache.k_scale.mul_(2.0 ** keys)
    p.check(inv_temp=2.0 ** (-3 - queries - keys), wide=wide)


def narrow_and_full(dtype, dim=64, page=16, kv=8):
    rng = np.random.default_rng(3)
    count = 13 * sms() // 8
    lengths = [int(x) for x in rng.integers(64, 129, count)]
    new = [int(rng.integers(1, 33)) if r % 3 else 64 for r in range(count)]
    return Rows(lengths, new, heads=4 * kv, kv=kv, dim=dim, page=page, dtype=dtype, lean=2.0, seed=4).other_powers()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_tiles_of_different_widths_give_the_same_bits_every_time(dtype):
    """Calls that overlap on several streams."""
    from stickbreaking_attention_b200 import sb_attn_cached
    p = narrow_and_full(dtype)
    first = p.run(v=p.own_v)
    t, n, ends = (torch.tensor(np.ascontiguousarray(x), dtype=torch.int32, device="cuda") for x in (p.tables, p.lengths, np.cumsum(p.new)))
    call = lambda: sb_attn_cached(p.q, p.cache, t, n, ends, v=p.own_v)  # noqa: E731
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for out in outs for a, b in zip(out, first))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_nan_in_one_tile_of_many(dtype):
    """NaN in values that some queries of a tile see, in tiles of many, narrow and full: the results of those queries, in that column, and no others."""
    p = narrow_and_full(dtype)
    clean_o, clean_rem = p.run()
    bad = torch.zeros_like(clean_o, dtype=torch.bool)
    first = np.cumsum(p.new) - p.new
    for r in range(1, len(p.lengths), 5):
        length, n, g = p.lengths[r], p.new[r], r % p.kv
        key = length - 1 - n // 2  # seen by the rows behind it
        p.cache.v.view(torch.uint8)[int(p.tables[r, key // p.page]), g, key % p.page, 9] = 127
        sees = key - (length - n) + 1
        bad[4 * g:4 * g + 4, first[r] + sees:first[r] + n, 9] = True
    assert bad.any()
    o, rem = p.run()
    assert o[bad].isnan().all() and torch.equal(o[~bad], clean_o[~bad]) and torch.equal(rem, clean_rem)
