"""The 8-bit paged cache on a B200: append, read-back, attention and page moves against plain implementations in
64 bits (tests/cache_ref.py), at the sizes and masks where they can go wrong."""
import ctypes
import math

import numpy as np
import pytest
import torch

import cache_ref as ref

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch.device("cuda", 0)


def _err():
    from minicpm5_mk import _lib
    e = ctypes.c_int32()
    return _lib.lib().mk_get_error(None, ctypes.byref(e)), e.value


def _gpu(dev, *ts):
    return [t.to(dev) for t in ts]


def _i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32)


# ---------------------------------------------------------------------------------------- attention
def _attend(dev, lens, n_new, n_q, n_kv, hd, page, seed, spare=3, strided=True, q_scale=1.0, max_len=None):
    from minicpm5_mk import ops
    need = sum(-(-int(n) // page) for n in lens)
    codes, scales = ref.pool(need + spare, n_kv, page, hd, seed)
    table = ref.tables(lens, page, need + spare, seed)
    # what no row may read: pages that no table lists, NaN as their scale
    idle = sorted(set(range(need + spare)) - set(table[table >= 0].tolist()))
    scales[idle] = math.nan
    cu = _i32(np.concatenate([[0], np.cumsum(n_new)]))
    T = int(cu[-1])
    g = torch.Generator().manual_seed(seed + 1)
    wide = (q_scale * torch.randn((T, n_q + 2, hd + 8 if strided else hd), generator=g)).to(BF)
    q = wide[:, 1:1 + n_q, :hd] if strided else wide[:, :n_q].contiguous()
    one = all(n == 1 for n in n_new)
    qd = wide.to(dev)[:, 1:1 + n_q, :hd] if strided else q.to(dev)
    o, lse = ops.attention_paged(qd, *_gpu(dev, codes, scales, table, _i32(lens)), cu_q=None if one else cu.to(dev),
                                 max_q=max(n_new), max_len=max_len, softmax_scale=1 / math.sqrt(hd))
    want, wl, av, err = ref.attend(q, codes, scales, table, lens, cu, 1 / math.sqrt(hd))
    assert _err() == (0, 0)
    _close(o, lse, want, wl, av, err)


def _close(o, lse, want, wl, av, err):
    o, lse = o.double().cpu(), lse.double().cpu()
    none = wl == -math.inf
    assert torch.equal(lse == -math.inf, none) and bool((o[none] == 0).all())
    # lse: the scores' f32 error (each moves lse by at most as much), 2^-20 for the exponentials and the sum
    assert bool(((lse - wl).abs()[~none] <= (err + 2.0 ** -20 * (1 + wl.abs()))[~none]).all())
    # out: the probabilities carry the scores' error twice over and are rounded to 11 bits before the product
    # (2^-11 each, 2^-10 allowed), the result once to bf16 (2^-9, 2^-8 allowed)
    tol = av * (2.0 ** -10 + 2 * err[..., None]) + want.abs() * 2.0 ** -8 + 1e-30
    assert bool(((o - want).abs() <= tol).all()), float(((o - want).abs() / tol).max())


@pytest.mark.parametrize("hd", [96, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("n_q,n_kv", [(16, 2), (4, 4), (12, 4), (4, 1)])
def test_attention_single_tokens(dev, hd, page, n_q, n_kv):
    lens = [1, 0, 2, page - 1, page, page + 1, 15, 17, 333]
    _attend(dev, lens, [1] * len(lens), n_q, n_kv, hd, page, 7 + hd + page + n_q)


@pytest.mark.parametrize("hd,page,n_q,n_kv", [(96, 16, 16, 2), (128, 64, 16, 2), (96, 32, 6, 2), (128, 128, 7, 7),
                                              (128, 32, 32, 1)])
def test_attention_ragged_chunks(dev, hd, page, n_q, n_kv):
    # chunks of one token, a whole prompt, more than a tile of rows, none at all, and an idle row
    lens, new = [1, 40, 64, 130, 257, 0, 300, 9], [1, 40, 3, 17, 70, 0, 0, 2]
    _attend(dev, lens, new, n_q, n_kv, hd, page, 31 + hd + n_q)


@pytest.mark.parametrize("hd,page,n_q,n_kv", [(96, 16, 16, 2), (128, 64, 16, 2), (96, 128, 12, 4)])
@pytest.mark.parametrize("top", [2, 4, 8, 9, 16, 33])
def test_attention_chunk_sizes(dev, hd, page, n_q, n_kv, top):
    """Chunks up to `top` tokens: every width of query tile, whole tiles and parts of them."""
    lens, new = [top, 200, 64, 0, 333, 1000], [top, 1, max(1, top // 2), 0, top, top - 1]
    _attend(dev, lens, new, n_q, n_kv, hd, page, 57 + hd + top)


@pytest.mark.parametrize("hd,page", [(96, 16), (128, 32), (128, 128)])
def test_attention_chunk_with_a_nan_scale_and_a_missing_page(dev, hd, page):
    """Wide tiles: a NaN scale shows in the queries that see its page, a missing page is reported, and what lies
    past a row's end (garbage codes, NaN scales) does not show."""
    from minicpm5_mk import ops
    lens, new, n_q, n_kv = [3 * page, 200, 150], [20, 30, 40], 16, 2
    need = sum(-(-n // page) for n in lens)
    codes, scales = ref.pool(need + 2, n_kv, page, hd, 4)
    table = ref.tables(lens, page, need + 2, 4)
    idle = sorted(set(range(need + 2)) - set(table[table >= 0].tolist()))
    scales[idle] = math.nan
    cu = _i32([0, 20, 50, 90])
    q = torch.randn((90, n_q, hd), generator=torch.Generator().manual_seed(1)).to(BF)
    want = ref.attend(q, codes, scales, table, lens, cu, 0.1)
    bad = scales.clone()
    bad[table[0, 2], 1, 1] = math.nan  # the last page of row 0, values of head 1: seen by the queries from 2 * page on
    o, lse = ops.attention_paged(*_gpu(dev, q, codes, bad, table, _i32(lens)), cu_q=cu.to(dev), max_q=40, max_len=3 * page,
                                 softmax_scale=0.1)
    hit = torch.zeros((90, n_q), dtype=torch.bool)
    hit[[t for t in range(20) if 3 * page - 20 + t >= 2 * page], 8:] = True
    assert o.isnan().all(-1).cpu().equal(hit) and o.isnan().any(-1).cpu().equal(hit)
    ok = ~hit
    _close(o.cpu()[ok], lse.cpu()[ok], *[w[ok] for w in want])
    t = table.clone()
    t[1, 0] = -1
    o, lse = ops.attention_paged(*_gpu(dev, q, codes, scales, t, _i32(lens)), cu_q=cu.to(dev), max_q=40, softmax_scale=0.1)
    assert _err() == (10, 0x500)
    keep = [i for i in range(90) if not 20 <= i < 50]
    _close(o[keep], lse[keep], *[w[keep] for w in want])
    assert bool(o[20:50].isfinite().all())


def test_attention_queries_before_the_first_key(dev):
    """More queries than tokens (a padded chunk): the first see nothing."""
    _attend(dev, [3, 0, 20], [5, 2, 4], 4, 2, 96, 16, 5)


@pytest.mark.parametrize("lens", [[5000], [1, 9000], [2049, 0, 4096, 12345]])
@pytest.mark.parametrize("hd,page", [(96, 64), (128, 128), (128, 16)])
def test_attention_long(dev, lens, hd, page):
    _attend(dev, lens, [1] * len(lens), 16, 2, hd, page, 11 + len(lens))


def test_attention_long_chunk(dev):
    _attend(dev, [3001, 700], [33, 2], 16, 2, 96, 64, 77)


def test_attention_large_scores(dev):
    """Scores of several hundred: no exponential overflows, and one key takes a row."""
    _attend(dev, [700, 64, 5], [1, 1, 1], 16, 2, 128, 64, 3, q_scale=40.0)


def test_attention_contiguous_queries_and_tight_bound(dev):
    _attend(dev, [100, 64], [1, 1], 8, 2, 96, 32, 21, strided=False, max_len=100)


def test_attention_many_rows(dev):
    lens = [(37 * i) % 90 for i in range(700)]
    _attend(dev, lens, [1] * 700, 4, 2, 96, 16, 8)


def test_attention_value_scales_far_apart(dev):
    """Pages whose value scales differ by 2^60, and one of all-zero values."""
    from minicpm5_mk import ops
    lens, page, hd = [128], 32, 96
    codes, scales = ref.pool(4, 2, page, hd, 9)
    table = ref.tables(lens, page, 4, 9)
    scales[table[0, 0], 1] *= 2.0 ** -60
    scales[table[0, 1], 1] = 0.0
    codes[table[0, 1].long(), 1] = 0
    scales[table[0, 2], 1] *= 2.0 ** 30
    q = torch.randn((1, 16, hd), generator=torch.Generator().manual_seed(1)).to(BF)
    o, lse = ops.attention_paged(*_gpu(dev, q, codes, scales, table, _i32(lens)), softmax_scale=0.1)
    _close(o, lse, *ref.attend(q, codes, scales, table, lens, [0, 1], 0.1))


def test_attention_nan_scale_shows(dev):
    """A page whose scale is NaN makes the heads that read it NaN, and no others."""
    from minicpm5_mk import ops
    lens, page, hd = [50, 50], 16, 128
    codes, scales = ref.pool(8, 2, page, hd, 4)
    table = ref.tables(lens, page, 8, 4)
    scales[table[0, 1], 0, 1] = math.nan   # keys of head 1, row 0
    scales[table[1, 0], 1, 0] = math.nan   # values of head 0, row 1
    q = torch.randn((2, 4, hd), generator=torch.Generator().manual_seed(1)).to(BF)
    o, lse = ops.attention_paged(*_gpu(dev, q, codes, scales, table, _i32(lens)), softmax_scale=0.1)
    bad = o.isnan().any(-1).cpu()
    assert bad.tolist() == [[False, False, True, True], [True, True, False, False]]
    assert o.isnan().all(-1).cpu().equal(bad)
    assert lse.isnan().cpu().tolist()[0] == [False, False, True, True]


def test_attention_zero_and_tiny_queries(dev):
    """Zero queries weigh all keys alike; queries near bf16's smallest do too, without a NaN."""
    from minicpm5_mk import ops
    lens, page, hd = [70, 70, 70], 32, 96
    codes, scales = ref.pool(9, 2, page, hd, 4)
    table = ref.tables(lens, page, 9, 4)
    q = torch.zeros((3, 4, hd), dtype=BF)
    q[1] = 1e-38
    q[2, :, ::2] = 1e-30
    q[2, :, 3] = 1.5
    o, lse = ops.attention_paged(*_gpu(dev, q, codes, scales, table, _i32(lens)), softmax_scale=0.1)
    _close(o, lse, *ref.attend(q, codes, scales, table, lens, [0, 1, 2, 3], 0.1))


def test_attention_offsets_past_32_bits(dev):
    """Pages more than 4 GiB into the pool."""
    from minicpm5_mk import ops
    page, hd, n_kv = 128, 128, 2
    pages = (1 << 32) // (2 * n_kv * page * hd) + 40
    lens = [300, 129]
    need = 5
    codes, scales = ref.pool(need, n_kv, page, hd, 6)
    table = ref.tables(lens, page, need, 6)
    big = torch.empty((pages, 2, n_kv, page, hd), dtype=torch.int8, device=dev)
    bs = torch.full((pages, 2, n_kv), math.nan, device=dev)
    big[pages - need:], bs[pages - need:] = codes.to(dev), scales.to(dev)
    far = torch.where(table >= 0, table + (pages - need), -1)
    q = torch.randn((2, 16, hd), generator=torch.Generator().manual_seed(1)).to(BF)
    o, lse = ops.attention_paged(q.to(dev), big, bs, *_gpu(dev, far, _i32(lens)), softmax_scale=0.1)
    _close(o, lse, *ref.attend(q, codes, scales, table, lens, [0, 1, 2], 0.1))
    # the same for append and read-back
    k = torch.randn((3, n_kv, hd), generator=torch.Generator().manual_seed(2)).to(BF)
    cu = _i32([0, 2, 3])
    ops.kv_append(*_gpu(dev, k, k), big, bs, *_gpu(dev, far, _i32(lens)), cu_new=cu.to(dev), max_new=2)
    ref.append(k, k, codes, scales, table, lens, cu)
    kk, vv = ops.kv_read(big, bs, *_gpu(dev, far, _i32([0, 0]), _i32([302, 130])), 302)
    for r, n in enumerate((302, 130)):
        a, b = ref.planes(codes, scales, table[r, :-(-n // page)].long())
        assert kk[r, :n].cpu().equal(a[:n].float().to(BF)) and vv[r, :n].cpu().equal(b[:n].float().to(BF))
    assert _err() == (0, 0)


def test_attention_on_another_stream(dev):
    from minicpm5_mk import ops
    lens, page, hd = [3000, 100], 64, 96
    codes, scales = ref.pool(49, 2, page, hd, 4)
    table = ref.tables(lens, page, 49, 4)
    q = torch.randn((2, 16, hd), generator=torch.Generator().manual_seed(1)).to(BF)
    args = _gpu(dev, q, codes, scales, table, _i32(lens))
    want = ref.attend(q, codes, scales, table, lens, [0, 1, 2], 0.1)
    torch.cuda.synchronize()
    got = []
    for s in (torch.cuda.Stream(dev), torch.cuda.Stream(dev)):
        with torch.cuda.stream(s):
            for _ in range(3):
                got.append(ops.attention_paged(*args, softmax_scale=0.1))
    torch.cuda.synchronize()
    for o, lse in got:
        _close(o, lse, *want)
        assert o.equal(got[0][0]) and lse.equal(got[0][1])  # the same bits each time


def test_attention_missing_page_is_reported(dev):
    """A table without a page that a row's length needs, or with an id out of range: the error word is set and the
    other rows are right."""
    from minicpm5_mk import ops
    lens, page, hd = [40, 40, 40], 16, 96
    codes, scales = ref.pool(9, 2, page, hd, 4)
    table = ref.tables(lens, page, 9, 4)
    q = torch.randn((3, 4, hd), generator=torch.Generator().manual_seed(1)).to(BF)
    want = ref.attend(q, codes, scales, table, lens, [0, 1, 2, 3], 0.1)
    for bad in (-1, 9, 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[1, 1] = bad
        o, lse = ops.attention_paged(*_gpu(dev, q, codes, scales, t, _i32(lens)), softmax_scale=0.1)
        st, e = _err()
        assert st == 10 and e == 0x500
        ok = [0, 2]
        _close(o[ok], lse[ok], *[w[ok] for w in want])
    assert _err() == (0, 0)


@pytest.mark.parametrize("hd,page,n_q,n_kv", [(96, 64, 16, 2), (128, 16, 16, 2), (96, 128, 2, 2), (128, 32, 10, 2)])
@pytest.mark.parametrize("top", [4096, 8192])
def test_attention_single_tokens_of_few_rows(dev, hd, page, n_q, n_kv, top):
    """Lengths around where the shares of eight CTAs begin and end, and up to where the launch changes its form."""
    lens = [0, 1, 127, 128, 129, 1023, 1024, 1025, 1151, 2047, top - 129, top][: 7 if top == 4096 else 12]
    _attend(dev, lens, [1] * len(lens), n_q, n_kv, hd, page, 5 + hd + n_q, max_len=top)


@pytest.mark.parametrize("case", [test_attention_large_scores, test_attention_contiguous_queries_and_tight_bound,
                                  test_attention_value_scales_far_apart, test_attention_nan_scale_shows,
                                  test_attention_zero_and_tiny_queries, test_attention_offsets_past_32_bits,
                                  test_attention_on_another_stream, test_attention_missing_page_is_reported])
def test_attention_single_tokens_as_chunks(dev, monkeypatch, case):
    """Single tokens given as chunks of one take another way through the library: the cases above hold there too."""
    from minicpm5_mk import ops
    plain = ops.attention_paged

    def chunks(q, *args, cu_q=None, **kw):
        each = torch.arange(q.shape[0] + 1, dtype=torch.int32, device=q.device)
        return plain(q, *args, cu_q=each if cu_q is None else cu_q, **kw)

    monkeypatch.setattr(ops, "attention_paged", chunks)
    case(dev)


@pytest.mark.parametrize("top", [1, 40])
def test_lengths_and_tokens_out_of_range_are_reported(dev, top):
    """Lengths past the table (up to the largest int) and token ranges past T read and write nothing outside; the
    other rows are right."""
    from minicpm5_mk import ops
    lens, page, hd = [60, 60, 60], 16, 96
    codes, scales = ref.pool(13, 2, page, hd, 4)
    table = ref.tables(lens, page, 13, 4)
    T = 3 * top
    q = torch.randn((T, 16, hd), generator=torch.Generator().manual_seed(1)).to(BF)
    cu = _i32([0, top, 2 * top, 3 * top])
    want = ref.attend(q, codes, scales, table, lens, cu, 0.1)
    one = dict(cu_q=cu.to(dev), max_q=top) if top > 1 else {}
    keep = list(range(top)) + list(range(2 * top, T))
    for bad in (65, 2 ** 31 - 1):
        o, lse = ops.attention_paged(*_gpu(dev, q, codes, scales, table, _i32([60, bad, 60])), **one, softmax_scale=0.1)
        assert _err() == (10, 0x500)
        _close(o[keep], lse[keep], *[w[keep] for w in want])
    for bad in ([0, top, 2 * top, 2 ** 31 - 1], [0, top, 2 * top, T + 1], [0, top, -5, T], [0, -2 ** 31, 2 * top, T]):
        o, lse = ops.attention_paged(*_gpu(dev, q, codes, scales, table, _i32(lens)), cu_q=_i32(bad).to(dev), max_q=top,
                                     softmax_scale=0.1)
        assert _err()[0] in (0, 10)
        if bad[1] == top:
            _close(o[:top], lse[:top], *[w[:top] for w in want])
    cd, sd = _gpu(dev, codes, scales)
    x = torch.ones((2, 2, hd), dtype=BF, device=dev)
    for ln, c in (([64, 2 ** 31 - 1, 0], [0, 1, 2, 2]), ([0, 0, 0], [0, 3, 3, 3]), ([0, 0, 0], [0, -1, 0, 2 ** 31 - 1])):
        ops.kv_append(x, x, cd, sd, *_gpu(dev, table, _i32(ln), _i32(c)), max_new=5)
        assert _err() == (10, 0x500)
    # (the last of them wrote row 1's token -1 .. 0 nowhere, and the pool is as it was)
    assert cd.cpu().equal(codes) and sd.cpu().equal(scales)
    k, v = ops.kv_read(cd, sd, *_gpu(dev, table, _i32([2 ** 31 - 1, 64, 60]), _i32([4, 4, 2 ** 31 - 1])), 8)
    assert _err() == (10, 0x500)
    assert not bool(k[:2].any()) and not bool(k[2, 4:].any())
    pool6 = cd[None].contiguous(), sd[None].contiguous()
    refs = torch.ones(13, dtype=torch.int32, device=dev)
    t, n, f = ops.kv_fork(*pool6, *_gpu(dev, table, _i32([60, 2 ** 31 - 1, 60])), refs, _i32([1, 1, 0, 2 ** 31 - 1]).to(dev))
    assert _err() == (10, 0x500) and n.cpu().tolist() == [64, 64, 60, 0]
    ops.kv_reserve(t, _i32([2 ** 31 - 1, 64, 60, 0]).to(dev), f, _i32([2 ** 31 - 1, 1, 0, 0]).to(dev), page)
    assert _err()[0] == 10


# ---------------------------------------------------------------------------------------- append, read
def _check_pool(codes, scales, got_codes, got_scales, ids):
    ids = [int(i) for i in ids]
    assert scales[ids].numpy().tobytes() == got_scales[ids].cpu().numpy().tobytes() or \
        torch.equal(torch.nan_to_num(scales[ids], nan=-1.0), torch.nan_to_num(got_scales[ids].cpu(), nan=-1.0))
    assert torch.equal(codes[ids], got_codes[ids].cpu())


@pytest.mark.parametrize("hd", [96, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_append_matches_the_definition(dev, hd, page):
    """Ragged appends onto empty, part-filled and full last pages; the codes and scales are equal bit for bit."""
    from minicpm5_mk import ops
    n_kv = 2
    lens = [0, 1, 3, page - 1, page, 2 * page + 5, 7, 0, page - 2]
    new = [1, 2 * page + 3, 4, 1, 1, page, 0, page, 3]
    total = [a + b for a, b in zip(lens, new)]
    pages = sum(-(-n // page) for n in total) + 2
    codes, scales = ref.pool(pages, n_kv, page, hd, 12)
    table = ref.tables(total, page, pages, 12)
    cu = _i32(np.concatenate([[0], np.cumsum(new)]))
    g = torch.Generator().manual_seed(3)
    # amplitudes from far below to far above what the pages hold, so that some scales grow and some do not
    amp = torch.logspace(-2, 2, int(cu[-1]))[:, None, None]
    wide = (torch.randn((int(cu[-1]), 7, hd + 8), generator=g) * amp).to(BF)
    wd = wide.to(dev)
    k, v = wide[:, 1:3, :hd], wide[:, 4:6, 8:]
    cd, sd = codes.to(dev), scales.to(dev)
    ops.kv_append(wd[:, 1:3, :hd], wd[:, 4:6, 8:], cd, sd, *_gpu(dev, table, _i32(lens), cu), max_new=max(new))
    ref.append(k, v, codes, scales, table, lens, cu)
    _check_pool(codes, scales, cd, sd, range(pages))  # whatever was not written stays
    assert _err() == (0, 0)


def test_append_token_by_token(dev):
    """One token at a time over several pages, values growing and shrinking: bit for bit, and near the input."""
    from minicpm5_mk import ops
    n_kv, hd, page, n = 2, 96, 16, 40
    codes, scales = ref.pool(7, n_kv, page, hd, 1)
    table = ref.tables([n, n], page, 7, 1)
    cd, sd, td = _gpu(dev, codes, scales, table)
    g = torch.Generator().manual_seed(3)
    x = (torch.randn((n, 2, 2, n_kv, hd), generator=g) * (1 + torch.arange(n) % 7)[:, None, None, None, None]).to(BF)
    for i in range(n):
        ops.kv_append(x[i, 0].to(dev), x[i, 1].to(dev), cd, sd, td, _i32([i, i]).to(dev))
        ref.append(x[i, 0], x[i, 1], codes, scales, table, [i, i], [0, 1, 2])
    _check_pool(codes, scales, cd, sd, table[table >= 0])
    k, v = ops.kv_read(cd, sd, td, *_gpu(dev, _i32([0, 0]), _i32([n, n])), n)
    for got, w in ((k, 0), (v, 1)):
        y = x[:, w].transpose(0, 1).double()
        # at most 7 growths of a page's scale: half a step each, of a step that is max / 127, and bf16's rounding
        top = torch.stack([y[:, i // page * page:min(n, (i // page + 1) * page)].abs().amax((1, 3)) for i in range(n)], 1)
        assert bool(((got.cpu().double() - y).abs() <= (4 / 127 + 2.0 ** -8) * top[..., None]).all())


def test_append_zeros_and_non_finite(dev):
    from minicpm5_mk import ops
    n_kv, hd, page = 2, 128, 16
    codes, scales = ref.pool(6, n_kv, page, hd, 1)
    lens, new = [0, 5, 3, 0], [4, 3, 6, 17]
    table = ref.tables([a + b for a, b in zip(lens, new)], page, 6, 1)
    cu = _i32(np.concatenate([[0], np.cumsum(new)]))
    x = torch.randn((30, 2, n_kv, hd), generator=torch.Generator().manual_seed(3)).to(BF)
    x[:4] = 0
    x[5, 0, 1, 7] = math.inf
    x[8, 1, 0, 127] = math.nan
    x[13:, 1] = -0.0
    cd, sd = codes.to(dev), scales.to(dev)
    xd = x.to(dev)
    ops.kv_append(xd[:, 0], xd[:, 1], cd, sd, *_gpu(dev, table, _i32(lens), cu), max_new=17)
    ref.append(x[:, 0], x[:, 1], codes, scales, table, lens, cu)
    _check_pool(codes, scales, cd, sd, range(6))
    assert int(scales.isnan().sum()) == 2
    # a page that reads as NaN stays so until it is begun anew
    again = torch.ones((4, n_kv, hd), dtype=BF)
    ops.kv_append(again.to(dev), again.to(dev), cd, sd, *_gpu(dev, table, _i32([4, 8, 9, 0])))
    ref.append(again, again, codes, scales, table, [4, 8, 9, 0], [0, 1, 2, 3, 4])
    _check_pool(codes, scales, cd, sd, range(6))
    assert int(sd.isnan().sum()) == 2
    ops.kv_append(again.to(dev), again.to(dev), cd, sd, *_gpu(dev, table, _i32([0, 0, 0, 0])))
    assert not bool(sd.isnan().any()) and _err() == (0, 0)


def test_read_ranges(dev):
    from minicpm5_mk import ops
    n_kv, hd, page = 3, 96, 16
    lens = [50, 17, 0, 33]
    codes, scales = ref.pool(10, n_kv, page, hd, 1)
    table = ref.tables(lens, page, 10, 1)
    args = _gpu(dev, codes, scales, table)
    for start, count, top in [([0, 0, 0, 0], lens, 50), ([3, 16, 0, 5], [40, 1, 0, 27], 40), ([49, 0, 0, 32], [1, 2, 0, 1], 5),
                              ([1, 2, 0, 3], [9, 9, 0, 9], 4)]:
        k, v = ops.kv_read(*args, *_gpu(dev, _i32(start), _i32(count)), top)
        for r in range(4):
            n = min(count[r], top)
            if n:
                a, b = ref.planes(codes, scales, table[r, :-(-lens[r] // page)].long())
                s = slice(start[r], start[r] + n)
                assert k[r, :n].cpu().equal(a[s].float().to(BF)) and v[r, :n].cpu().equal(b[s].float().to(BF))
            assert not bool(k[r, n:].any()) and not bool(v[r, n:].any())
    assert _err() == (0, 0)


def test_append_of_more_tokens_than_announced_is_reported(dev):
    """max_new bounds a row's new tokens: pages past those that so many can touch are left alone, and the error word
    says so.  40 tokens from position 3 touch three pages of 16, 18 may as well, 2 touch two at most."""
    from minicpm5_mk import ops
    codes, scales = ref.pool(5, 2, 16, 96, 1)
    table = ref.tables([64], 16, 5, 1)
    x = torch.randn((40, 2, 96), generator=torch.Generator().manual_seed(3)).to(BF).to(dev)
    cd, sd = codes.to(dev), scales.to(dev)
    ops.kv_append(x, x, cd, sd, *_gpu(dev, table, _i32([3]), _i32([0, 40])), max_new=2)
    assert _err() == (10, 0x500)
    for p in (*table[0, 2:].tolist(), *sorted(set(range(5)) - set(table[0].tolist()))):
        assert cd[p].cpu().equal(codes[p]) and sd[p].cpu().equal(scales[p])
    for bound in (18, 40):
        cd, sd = codes.to(dev), scales.to(dev)
        ops.kv_append(x, x, cd, sd, *_gpu(dev, table, _i32([3]), _i32([0, 40])), max_new=bound)
        c, s = codes.clone(), scales.clone()
        ref.append(x.cpu(), x.cpu(), c, s, table, [3], [0, 40])
        _check_pool(c, s, cd, sd, range(5))
    assert _err() == (0, 0)


@pytest.mark.parametrize("rows", [2, 40])
def test_decoding_step_in_a_graph(dev, rows):
    """Pages reserved, keys appended, attention and scores of one step captured once: each replay gives what the calls
    give outside."""
    from minicpm5_mk import ops
    page, hd, n_kv, steps = 16, 96, 2, 20
    lens = [(7 * r) % 50 for r in range(rows)]
    width, pages = 5, 5 * rows + 1
    codes, scales = ref.pool(pages, n_kv, page, hd, 3)
    start = ref.tables(lens, page, pages, 3)
    table = torch.full((rows, width), -1, dtype=torch.int32)
    table[:, :start.shape[1]] = start
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[table[table >= 0].long()] = 1
    g = torch.Generator().manual_seed(2)
    x = torch.randn((steps + 3, rows, 12, hd), generator=g).to(BF).to(dev)
    logits = torch.randn((steps + 3, rows, 5000), generator=g).to(dev)
    ids = torch.randint(0, 5000, (rows,), generator=g, dtype=torch.int32).to(dev)

    def state():
        return [t.clone() for t in _gpu(dev, codes, scales, table, _i32(lens), refs)]

    def step(st, xs, lg):
        cd, sd, t, n, f = st
        ops.kv_reserve(t, n, f, None, page)
        ops.kv_append(xs[:, 8:10], xs[:, 10:12], cd, sd, t, n)
        n += 1
        return (*ops.attention_paged(xs[:, :8], cd, sd, t, n, softmax_scale=0.1), *ops.token_logprobs(lg, ids, 3))

    there, here = state(), state()
    xs, lg = x[0].clone(), logits[0].clone()
    side = torch.cuda.Stream(dev)
    with torch.cuda.stream(side):
        step(state(), xs, lg)  # outside a capture first
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            got = step(there, xs, lg)
    for t, w in zip(there, state()):
        t.copy_(w)
    for i in range(steps):
        xs.copy_(x[i])
        lg.copy_(logits[i])
        graph.replay()
        for a, b in zip(got, step(here, x[i], logits[i])):
            assert a.equal(b)
    for a, b in zip(there, here):
        assert a.equal(b)
    assert _err() == (0, 0)


def test_append_without_a_page_is_reported(dev):
    from minicpm5_mk import ops
    codes, scales = ref.pool(4, 2, 16, 96, 1)
    table = ref.tables([16, 16], 16, 4, 1)
    cd, sd = codes.to(dev), scales.to(dev)
    x = torch.ones((2, 2, 96), dtype=BF, device=dev)
    ops.kv_append(x, x, cd, sd, *_gpu(dev, table, _i32([16, 0])))  # row 0 is full
    assert _err() == (10, 0x500)
    ref.append(x.cpu()[1:], x.cpu()[1:], codes, scales, table[1:], [0], [0, 1])
    _check_pool(codes, scales, cd, sd, range(4))


# ---------------------------------------------------------------------------------------- page moves
def _rows(seed, rows, page, top, pages, extra=1):
    r = np.random.RandomState(seed)
    lens = r.randint(0, top + 1, size=rows)
    lens[0], lens[-1] = 0, top
    table = ref.tables(lens, page, pages, seed, width=-(-top // page) + extra)
    return r, lens, table


@pytest.mark.parametrize("rows,new_rows,page,top,layers", [(1, 1, 16, 5, 1), (5, 9, 16, 70, 2), (40, 64, 32, 200, 3),
                                                         (300, 1500, 16, 40, 1), (8, 3, 128, 300, 2)])
def test_fork(dev, rows, new_rows, page, top, layers):
    from minicpm5_mk import ops
    pages = rows * (-(-top // page)) + 2 * new_rows + 3
    r, lens, table = _rows(rows, rows, page, top, pages)
    codes, scales = ref.pool(pages, 2, page, 96, 2, layers)
    parents = r.randint(-1, rows, size=new_rows).astype(np.int32)
    refs = torch.bincount(table[table >= 0].long(), minlength=pages).int()
    cd, sd = codes.to(dev), scales.to(dev)
    t, n, f = ops.kv_fork(cd, sd, *_gpu(dev, table, _i32(lens), refs, _i32(parents)))
    wt, wn, wf = ref.fork(codes, scales, table, lens, parents, pages)
    assert t.cpu().equal(wt) and n.cpu().equal(wn) and f.cpu().equal(wf)
    assert cd.cpu().equal(codes) and sd.cpu().equal(scales)
    # the next tokens' pages, then a second fork from the shared rows
    add = _i32(r.randint(0, 2, size=new_rows))
    ops.kv_reserve(t, n, f, add.to(dev), page)
    ref.reserve(wt, wn, wf, add, page)
    assert t.cpu().equal(wt) and f.cpu().equal(wf)
    parents = r.randint(-1, new_rows, size=new_rows).astype(np.int32)
    t, n, f = ops.kv_fork(cd, sd, t, n, f, _i32(parents).to(dev))
    wt, wn, wf = ref.fork(codes, scales, wt, wn, parents, pages)
    assert t.cpu().equal(wt) and n.cpu().equal(wn) and f.cpu().equal(wf)
    assert cd.cpu().equal(codes) and sd.cpu().equal(scales)
    assert _err() == (0, 0)


def test_fork_frees_what_is_dropped(dev):
    from minicpm5_mk import ops
    codes, scales = ref.pool(8, 2, 16, 96, 2, 2)
    table = ref.tables([40, 40], 16, 8, 2)
    cd, sd = codes.to(dev), scales.to(dev)
    t, n, f = ops.kv_fork(cd, sd, *_gpu(dev, table, _i32([40, 40]), _i32([1] * 8), _i32([-1, 1])))
    assert f.cpu().tolist() == [int(p in table[1].tolist()) for p in range(8)]
    assert t.cpu()[0].tolist() == [-1] * 3 and n.cpu().tolist() == [0, 40]
    t, n, f = ops.kv_fork(cd, sd, t, n, f, torch.empty(0, dtype=torch.int32, device=dev))
    assert t.shape == (0, 3) and not bool(f.any())
    assert cd.cpu().equal(codes) and _err() == (0, 0)


def test_no_free_page_is_reported(dev):
    from minicpm5_mk import ops
    codes, scales = ref.pool(3, 2, 16, 96, 2, 1)
    table = ref.tables([20], 16, 3, 2, width=2)
    args = _gpu(dev, codes, scales, table, _i32([20]), _i32([1, 1, 1]))
    t, n, f = ops.kv_fork(*args, _i32([0, 0, 0]).to(dev))  # two copies asked, one page free
    assert _err() == (10, 0x501)
    assert t.cpu()[1, 1] >= 0 and t.cpu()[2, 1] == -1
    ops.kv_reserve(t, n, f, _i32([13, 0, 0]).to(dev), 16)  # past the table's width
    assert _err() == (10, 0x501)
    ops.kv_fork(*args, _i32([1]).to(dev))  # no such row
    assert _err() == (10, 0x500)


def test_reserve_many_and_again(dev):
    from minicpm5_mk import ops
    for rows, page, pages in ((3, 16, 40), (8192, 16, 40000), (1200, 128, 3000)):
        r = np.random.RandomState(rows)
        lens = r.randint(0, 2 * page, size=rows)
        table = ref.tables(lens, page, pages, rows, width=5)
        refs = torch.bincount(table[table >= 0].long(), minlength=pages).int()
        add = _i32(r.randint(0, 2 * page, size=rows) if rows < 2000 else r.randint(0, 20, size=rows))
        t, n, f = _gpu(dev, table, _i32(lens), refs)
        for _ in range(2):  # a second call finds the pages there
            ops.kv_reserve(t, n, f, add.to(dev), page)
            if _ == 0:
                ref.reserve(table, lens, refs, add, page)
            assert t.cpu().equal(table) and f.cpu().equal(refs)
        assert _err() == (0, 0)


@pytest.mark.parametrize("pages,live", [(1, 1), (5, 0), (64, 64), (1000, 400), (1025, 1), (5000, 2600)])
def test_compact(dev, pages, live):
    from minicpm5_mk import ops
    r = np.random.RandomState(pages)
    ids = r.permutation(pages)[:live]
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[torch.from_numpy(ids).long()] = _i32(r.randint(1, 4, size=live))
    table = torch.full((max(1, -(-live // 3)), 4), -1, dtype=torch.int32)
    for i, p in enumerate(ids):
        table[i // 3, i % 3] = int(p)
    codes, scales = ref.pool(pages, 1, 16, 96, 2, 2)
    cd, sd = codes.to(dev), scales.to(dev)
    for _ in range(2):  # again from the same tables: the same result
        t, f, used = ops.kv_compact(cd, sd, *_gpu(dev, table, refs))
    wt, wf, wu = ref.compact(codes, scales, table, refs)
    assert t.cpu().equal(wt) and f.cpu().equal(wf) and int(used) == wu
    assert cd.cpu().equal(codes) and sd.cpu().equal(scales)
    assert _err() == (0, 0)


# ---------------------------------------------------------------------------------------- refusals
def test_refusals(dev):
    from minicpm5_mk import _lib, ops
    codes, scales = _gpu(dev, *ref.pool(4, 2, 16, 96, 1))
    table, lens = torch.zeros((2, 2), dtype=torch.int32, device=dev), torch.ones(2, dtype=torch.int32, device=dev)
    q = torch.zeros((2, 4, 96), dtype=BF, device=dev)
    ok = dict(q=q, codes=codes, scales=scales, block_table=table, lens=lens)
    ops.attention_paged(**ok)
    for change in (dict(q=q.float()), dict(q=q[..., :64]), dict(q=q.cpu()), dict(codes=codes[0]), dict(scales=scales[:2]),
                   dict(scales=scales.double()), dict(lens=lens[:1]), dict(lens=lens.long()), dict(block_table=table[0]),
                   dict(block_table=table.T), dict(q=q[:1]), dict(cu_q=lens), dict(q=q.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            ops.attention_paged(**{**ok, **change})
    for change in (dict(q=torch.zeros((2, 3, 96), dtype=BF, device=dev)),               # 3 query heads over 2
                   dict(q=torch.zeros((2, 4, 100), dtype=BF, device=dev)[..., 2:98]),   # not 16-byte aligned
                   dict(max_len=-1)):
        with pytest.raises(_lib.MkError):
            ops.attention_paged(**{**ok, **change})
    x = torch.zeros((2, 2, 96), dtype=BF, device=dev)
    with pytest.raises(ValueError):
        ops.kv_append(x, x[:1], codes, scales, table, lens)
    with pytest.raises(ValueError):
        ops.kv_append(x, x.half(), codes, scales, table, lens)
    with pytest.raises(_lib.MkError):  # page of 24 tokens
        ops.kv_append(x, x, torch.zeros((4, 2, 2, 24, 96), dtype=torch.int8, device=dev), scales, table, lens)
    with pytest.raises(_lib.MkError):  # head size 64
        ops.kv_read(torch.zeros((4, 2, 2, 16, 64), dtype=torch.int8, device=dev), scales, table, lens, lens, 4)
    with pytest.raises(_lib.MkError):
        ops.kv_reserve(table, lens, lens, None, 20)
    pool6 = codes[None].contiguous(), scales[None].contiguous()
    refs = torch.zeros(4, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError):
        ops.kv_fork(codes, scales, table, lens, refs, lens)
    with pytest.raises(ValueError):
        ops.kv_fork(*pool6, table, lens, refs[:3], lens)
    with pytest.raises(ValueError):
        ops.kv_compact(*pool6, table, refs.long())
    with pytest.raises(_lib.MkError):  # more rows than a call takes
        ops.kv_fork(*pool6, table, lens, refs, torch.zeros(8193, dtype=torch.int32, device=dev))
    assert _err() == (0, 0)


def test_nothing_to_do(dev):
    from minicpm5_mk import ops
    codes, scales = _gpu(dev, *ref.pool(4, 2, 16, 96, 1))
    none, table = torch.zeros(0, dtype=torch.int32, device=dev), torch.zeros((0, 3), dtype=torch.int32, device=dev)
    x = torch.zeros((0, 2, 96), dtype=BF, device=dev)
    before = codes.clone()
    ops.kv_append(x, x, codes, scales, table, none)
    o, lse = ops.attention_paged(torch.zeros((0, 4, 96), dtype=BF, device=dev), codes, scales, table, none)
    assert o.shape == (0, 4, 96) and lse.shape == (0, 4)
    k, v = ops.kv_read(codes, scales, table, none, none, 3)
    assert k.shape == (0, 3, 2, 96)
    ops.kv_reserve(table, none, torch.zeros(4, dtype=torch.int32, device=dev), None, 16)
    assert codes.equal(before) and _err() == (0, 0)
