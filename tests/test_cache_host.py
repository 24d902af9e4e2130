"""CPU checks of the 8-bit paged cache: refusals of the C ABI and of the Python layer, sizes, the oracle's own arithmetic."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import cache_oracle as orc


@pytest.fixture(scope="module")
def lib():
    from stickbreaking_attention_b200 import build, _lib
    build.build()
    return _lib.lib()


def blocks_params(**kw):  # its addresses are never followed: every call below is refused or has nothing to do
    from stickbreaking_attention_b200._lib import SbBlocksParams
    p = SbBlocksParams(requests=2, width=4, pages=8, page_tokens=16, tokens=5, n_pieces=4, table_stride=4)
    for name in ("lengths", "new_tokens", "free_count", "tables", "free_pages", "lengths_out", "free_count_out", "ends", "slots", "pieces", "status"):
        setattr(p, name, 4096)
    for k, v in kw.items():
        setattr(p, k, v)
    return ctypes.byref(p)


@pytest.mark.parametrize("change, code", [
    (dict(requests=-1), -1), (dict(width=-1), -1), (dict(pages=-1), -1), (dict(tokens=-1), -1), (dict(page_tokens=24), -1), (dict(page_tokens=0), -1),
    (dict(table_stride=3), -1), (dict(n_pieces=3), -1), (dict(requests=2049, n_pieces=9000), -3), (dict(width=1 << 27, table_stride=1 << 27), -3),
    (dict(tokens=(1 << 30) + 1, n_pieces=1 << 30), -3), (dict(lengths=None), -2), (dict(new_tokens=None), -2), (dict(free_count=None), -2), (dict(tables=None), -2),
    (dict(free_pages=None), -2), (dict(lengths_out=None), -2), (dict(free_count_out=None), -2), (dict(ends=None), -2), (dict(slots=None), -2),
    (dict(pieces=None), -2), (dict(pieces=4100), -5), (dict(status=None), -2)])
def test_blocks_refusals(lib, change, code):
    assert lib.sbattn_cache_blocks(blocks_params(**change)) == code


def cache_params(**kw):
    from stickbreaking_attention_b200._lib import SbCacheParams, SbMat, SbVec
    m = SbMat(4096, 0, 640, 64)
    p = SbCacheParams(dtype=0, heads=4, kv_heads=2, head_dim=64, row=64, page_tokens=16, pages=3, tokens=10, requests=2, width=2, n_pieces=4, inv_temp=0.1,
                      k_stride=2048, v_stride=2048, k_scale_stride=2, v_scale_stride=2, q=m, k=m, v=m, o=m, rem=SbVec(4096, 0, 10, 1), table_stride=2)
    for name in ("k_codes", "v_codes", "k_scale", "v_scale", "pieces", "tables", "lengths", "ends", "workspace", "status"):
        setattr(p, name, 4096)
    p.workspace_bytes = 1 << 40
    for k, v in kw.items():
        setattr(p, k, v)
    return ctypes.byref(p)


COMMON = [(dict(dtype=5), -1), (dict(kv_heads=-1), -1), (dict(head_dim=0), -1), (dict(head_dim=129, row=128), -3), (dict(row=128), -1), (dict(row=32), -1),
          (dict(page_tokens=48), -1), (dict(pages=0), -1), (dict(tokens=-1), -1), (dict(k_codes=None), -2), (dict(v_codes=None), -2), (dict(k_scale=None), -2),
          (dict(v_scale=None), -2), (dict(status=None), -2), (dict(k_stride=2047), -1), (dict(v_stride=1024), -1), (dict(k_scale_stride=1), -1),
          (dict(v_scale_stride=0), -1), (dict(k_codes=4104), -5), (dict(v_stride=2056), -5)]


@pytest.mark.parametrize("change, code", COMMON + [(dict(n_pieces=-1), -1), (dict(pieces=None), -2), (dict(pieces=4104), -5), (dict(n_pieces=1 << 30, kv_heads=4), -3)])
def test_append_refusals(lib, change, code):
    assert lib.sbattn_cache_append(cache_params(**change)) == code


@pytest.mark.parametrize("change, code", COMMON + [
    (dict(heads=3), -1), (dict(heads=-2), -1), (dict(kv_heads=0), -1), (dict(requests=-1), -1), (dict(requests=2049), -3), (dict(width=1 << 27, table_stride=1 << 27), -3),
    (dict(table_stride=1), -1), (dict(lengths=None), -2), (dict(tables=None), -2), (dict(ends=None, tokens=1), -1)])
def test_attend_refusals(lib, change, code):
    assert lib.sbattn_cached_fwd(cache_params(**change)) == code


def test_nothing_to_do(lib):
    assert lib.sbattn_cache_append(None) == -2 and lib.sbattn_cached_fwd(None) == -2 and lib.sbattn_cache_blocks(None) == -2
    assert lib.sbattn_cache_append(cache_params(n_pieces=0)) == 0
    assert lib.sbattn_cache_append(cache_params(tokens=0)) == 0
    assert lib.sbattn_cached_fwd(cache_params(tokens=0)) == 0
    assert lib.sbattn_cached_fwd(cache_params(heads=0)) == 0


def test_workspace_is_asked_for(lib):
    need = ctypes.c_size_t()
    assert lib.sbattn_cached_workspace_bytes(cache_params(), ctypes.byref(need)) == 0
    if need.value:
        assert lib.sbattn_cached_fwd(cache_params(workspace=None)) == -4
        assert lib.sbattn_cached_fwd(cache_params(workspace_bytes=need.value - 1)) == -4
        assert lib.sbattn_cached_fwd(cache_params(workspace=4096 + 16)) == -4


def test_pieces_bound(lib):
    """The bound holds for every way to share tokens out, and is reached."""
    rng = np.random.default_rng(0)
    for page in (16, 32):
        for _ in range(300):
            R, T = int(rng.integers(1, 8)), int(rng.integers(0, 90))
            cut = np.sort(rng.integers(0, T + 1, R - 1))
            new = np.diff(np.concatenate([[0], cut, [T]]))
            at = rng.integers(0, page, R)
            used = sum(-(-(a + n) // page) - a // page for a, n in zip(at, new) if n)
            assert used <= lib.sbattn_cache_pieces(R, T, page) == orc.pieces_bound(R, T, page)
    assert lib.sbattn_cache_pieces(3, 3, 16) == 3 and lib.sbattn_cache_pieces(1, 18, 16) == 3 and lib.sbattn_cache_pieces(0, 0, 16) == 0


def test_oracle_codes():
    v = orc.VALUES
    assert np.nanmax(v) == 448 and v[1] == 2.0 ** -9
    x = torch.randn(20000, generator=torch.Generator().manual_seed(0)).double() * torch.exp(3 * torch.randn(20000, generator=torch.Generator().manual_seed(1)).double())
    x = x.clamp(-448, 448).float()
    assert (torch.from_numpy(orc.to_code(x.double().numpy())) == x.to(torch.float8_e4m3fn).view(torch.uint8)).all()
    mid = (v[:126] + v[1:127]) / 2  # ties go to the even code
    assert (orc.to_code(mid) % 2 == 0).all()
    assert orc.scale_for(448.0) == 1.0 and orc.scale_for(449.0) == 2.0 and orc.scale_for(0.0) == 2.0 ** -118


def test_refused_without_cuda():
    from stickbreaking_attention_b200 import SbCache, sb_attn_cached, sb_cache, sb_cache_append, sb_cache_blocks
    c = sb_cache(2, 2, 50, 16, device="cpu")
    assert c.k.shape == (2, 2, 16, 64) and c.k.dtype == torch.float8_e4m3fn and c.k_scale.shape == (2, 2)
    q, i = torch.randn(2, 3, 50), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        sb_attn_cached(q, c, i.view(3, 1), i)
    with pytest.raises(RuntimeError, match="CUDA"):
        sb_cache_append(q, q, c, torch.zeros(1, 4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        sb_cache_blocks(i, i, i.view(3, 1), i, i[:1], 16, 3)
    for bad in (dict(head_dim=129), dict(head_dim=0), dict(page_tokens=48)):
        with pytest.raises(ValueError):
            sb_cache(**{**dict(pages=2, heads=2, head_dim=50, page_tokens=16, device="cpu"), **bad})


@pytest.mark.parametrize("wide", [0, 1, 2])
@pytest.mark.parametrize("current", [False, True])
def test_oracle_rows(wide, current):
    """The oracle of all rows at once is the one of single rows."""
    rng = np.random.default_rng(wide)
    for L, n in ((1, 1), (40, 7), (9, 9), (130, 1)):
        q, k, v, own = (rng.normal(0, 2, (x, 20)) for x in (n, L, L, n))
        for a, b in zip(orc.attend(q, k, v, n, 0.3, current, own, wide), orc.attend_rows(q, k, v, n, 0.3, current, own, wide)):
            assert a.shape == b.shape and np.allclose(a, b, rtol=1e-9, atol=1e-300)


def test_oracle_tiles():
    """Every step of every tile is dealt to one block, in order."""
    lengths, new = [1000, 1, 300, 90, 4000], [70, 1, 300, 0, 33]
    for blocks in (1, 3, 7, 148):
        dealt = orc.tiles_of_blocks(lengths, new, 3, 4, blocks)
        assert len(dealt) == blocks
        for tile in (256, 128):
            steps = sum(max(1, -(-(t - n + (min(c + tile, 4 * n) - 1) // 4) // 128)) for t, n in zip(lengths, new) for c in range(0, 4 * n, tile)) * 3
            assert sum(s for b in orc.tiles_of_blocks(lengths, new, 3, 4, blocks, tile=tile) for _, s in b) == steps
