"""GPU: the paged KV cache's append and the attention of one new token, against plain forms in 64 bits."""
import pytest
import torch

from tests.serving_reference import attend, attend_bounds, close, rows_of, turn, turn_bound

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def _pool(gen, dtype, lens, room, page, H, D, heads=True, spare=3, fill=float("nan")):
    """A pool in which every sequence has its own pages, in a random order, filled up to its length; the rest is `fill`."""
    B = len(lens)
    need = max(1, -(-(max(lens) + room) // page))
    pages = B * need + spare
    table = torch.randperm(pages, generator=gen, device=DEV)[: B * need].view(B, need).int()
    caches = []
    for _ in range(2):
        x = torch.full((pages, H, page, D) if heads else (pages, page, H, D), fill, device=DEV, dtype=dtype)
        x = x.transpose(1, 2) if heads else x
        for b, n in enumerate(lens):
            j = torch.arange(n, device=DEV)
            x[table[b, j // page].long(), j % page] = torch.randn(n, H, D, generator=gen, device=DEV).to(dtype)
        caches.append(x)
    return caches, table, torch.tensor(lens, dtype=torch.int32, device=DEV)


def _rand(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device=DEV).to(dtype)


def _check_decode(o, lse, q, caches, table, lens, scale, depth=None, turned=None, seen=None):
    """turned: (rotary, positions).  Keys are taken from the cache as it is now."""
    q64 = q.double()
    if turned is not None:
        rotary, at = turned
        q64 = turn(q64, at[:, None], rotary.inv_freq, rotary.interleaved, rotary.scale)
    for b, n in enumerate(lens):
        keys, values = (rows_of(c, table[b], n).double() for c in caches)
        if depth is not None:
            kd, vd = (x[b].double() if seen is None else x[b, : int(seen[b])].flatten(0, 1).double() for x in depth)
            keys, values = torch.cat([keys, kd]), torch.cat([values, vd])
        want_o, want_lse, size, mass = attend(q64[b], keys, values, scale)
        tol_o, tol_lse = attend_bounds(want_o, want_lse, size, mass, q.shape[-1], q.dtype, turned is not None)
        close(o[b], want_o, tol_o, f"o of sequence {b}")
        close(lse[b], want_lse, tol_lse, f"lse of sequence {b}")


DECODE = [  # dtype, lengths, H, G, D, L, page, heads
    (BF, [0], 1, 1, 64, 0, 1, True),
    (BF, [1], 1, 1, 64, 0, 16, True),
    (HF, [1, 0, 2], 2, 3, 128, 1, 5, False),
    (BF, [16, 17, 15, 31], 3, 4, 128, 7, 16, True),
    (HF, [256], 4, 1, 64, 4, 16, True),
    (BF, [1000, 3, 0, 511, 64], 5, 8, 128, 11, 24, False),
    (HF, [777, 778, 1, 65], 2, 9, 64, 3, 8, True),
    (BF, [300, 40], 1, 20, 128, 0, 64, False),
    (BF, [5000], 2, 4, 128, 32, 64, True),
    (HF, [20000, 1], 1, 2, 64, 1, 128, True),
    (BF, list(range(0, 290, 2)), 2, 2, 64, 5, 32, True),       # more sequences than a CTA has threads
    (BF, [33], 200, 1, 64, 2, 256, False),
    # more heads than CTAs: the work is divided evenly, whatever it is made of
    (HF, [(37 * i) % 301 for i in range(80)], 5, 3, 64, 4, 16, True),
    (BF, [(53 * i) % 900 for i in range(70)], 5, 4, 128, 7, 64, True),
    (BF, [0, 1, 15, 16, 17, 4000] * 12, 6, 2, 128, 0, 24, False),
    (HF, [2500, 0, 3, 900], 5, 9, 128, 2, 32, True),           # few heads, too long for clusters
    (BF, [9000, 8999], 8, 8, 64, 11, 256, True),
    (BF, [1] * 1000, 3, 1, 64, 0, 8, True),
    # more sequences than a CTA has threads, in units of single warps, of which many have none
    (BF, [(61 * i) % 198 for i in range(299)], 2, 2, 128, 1, 16, True),
    (HF, [(7 * i) % 90 for i in range(700)], 3, 1, 64, 3, 64, False),
    # just within what clusters are given, and beyond it
    (BF, [1530, 0, 700, 1531] * 9, 5, 2, 64, 7, 24, False),
    (HF, [2900, 2901] * 18, 5, 4, 64, 0, 32, True),
    (BF, [2700, 100, 2730, 5], 8, 4, 128, 16, 64, True),
    (BF, [12000, 11999], 8, 8, 64, 11, 256, True),
]


@pytest.mark.parametrize("dtype,lens,H,G,D,L,page,heads", DECODE)
def test_decode(built_library, dtype, lens, H, G, D, L, page, heads):
    """Rows behind a sequence's end, pages of nobody and whole unused pages hold NaN."""
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(len(lens) + H + L)
    B = len(lens)
    caches, table, n = _pool(gen, dtype, lens, 5, page, H, D, heads)
    q = _rand(gen, dtype, B, G, H, D)
    depth = tuple(_rand(gen, dtype, B, L, H, D) for _ in range(2)) if L else None
    kw = dict(cached_k=depth[0], cached_v=depth[1]) if L else {}
    o, lse = M.paged_moda_decode(q, *caches, table, n, **kw, moda_group_num=G, need_lse=True)
    _check_decode(o, lse, q, caches, table, lens, D ** -0.5, depth)
    again = M.paged_moda_decode(q, *caches, table, n, **kw, moda_group_num=G, need_lse=True)
    assert torch.equal(o, again[0]) and torch.equal(lse, again[1])
    assert M.device_status() == 0


@pytest.mark.parametrize("dtype,lens,H,G,D,L,page,heads", DECODE)
@pytest.mark.parametrize("interleaved,rot", [(False, 64), (True, 32)])
def test_step(built_library, dtype, lens, H, G, D, L, page, heads, interleaved, rot):
    """With the token's own key and value, turned, appended and recorded."""
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(len(lens) + H + L + 1)
    B = len(lens)
    caches, table, n = _pool(gen, dtype, lens, 1, page, H, D, heads)
    before = [c.clone() for c in caches]
    q, k, v = _rand(gen, dtype, B, G, H, D), _rand(gen, dtype, B, 1, H, D), _rand(gen, dtype, B, 1, H, D)
    rotary = M.Rotary(M.rotary_frequencies(rot, device=DEV)[0], interleaved, 1.1)
    depth = tuple(_rand(gen, dtype, B, L + 2, H, D) for _ in range(2))
    kw = dict(cached_k=depth[0][:, :L], cached_v=depth[1][:, :L], record_k=depth[0][:, L : L + 1], record_v=depth[1][:, L : L + 1])
    was = [x.clone() for x in depth]
    o, lse = M.paged_moda_decode(q, *caches, table, n, k, v, **kw, rotary=rotary, moda_group_num=G, need_lse=True)
    _check_decode(o, lse, q, caches, table, [x + 1 for x in lens], D ** -0.5, [x[:, :L] for x in depth] if L else None, (rotary, n.long()))
    want = turn(k.double(), n.long()[:, None], rotary.inv_freq, interleaved, 1.1)
    at = torch.arange(B, device=DEV)
    pages, slots = table[at, n.long() // page].long(), n.long() % page
    new_k, new_v = caches[0][pages, slots], caches[1][pages, slots]
    close(new_k[:, None], want, turn_bound(k.double(), want, rot, interleaved, 1.1, dtype), "the key's row")
    assert torch.equal(new_v[:, None], v)
    assert torch.equal(depth[0][:, L], new_k) and torch.equal(depth[1][:, L], new_v)
    for c, old, new in zip(caches, before, (new_k, new_v)):            # nothing else has been written
        old[pages, slots] = new
        assert torch.equal(c.view(torch.int16), old.view(torch.int16))
    for x, old in zip(depth, was):
        assert torch.equal(x[:, :L], old[:, :L]) and torch.equal(x[:, L + 1], old[:, L + 1])
    assert n.tolist() == lens and M.device_status() == 0


APPEND = [  # dtype, T, held, lengths, H, D, page, heads, rot, interleaved
    (BF, 1, [0], [1], 1, 64, 1, True, 64, False),
    (HF, 1, [5, 0, 64, 63], [1, 1, 1, 1], 8, 128, 64, True, 128, False),
    (BF, 7, [3, 0, 11], [7, 0, 4], 3, 128, 5, False, 96, True),
    (HF, 130, [0, 17], [130, 129], 2, 64, 16, True, 16, False),
    (BF, 33, [1], None, 20, 64, 24, False, 0, False),
    (BF, 1500, [0, 100, 7], [1500, 1, 777], 4, 128, 64, True, 64, True),
    (HF, 2, list(range(150)), None, 1, 64, 8, True, 48, True),
    (BF, 61, [0, 9, 64], [61, 3, 0], 1, 128, 16, True, 128, False),           # two and four tokens a warp
    (HF, 31, [5, 1, 0, 77, 3], [31, 30, 1, 0, 17], 1, 64, 24, False, 64, True),
    (BF, 3, [7] * 9, [1, 2, 3] * 3, 2, 64, 5, True, 32, False),
]


@pytest.mark.parametrize("dtype,T,held,lengths,H,D,page,heads,rot,interleaved", APPEND)
def test_append(built_library, dtype, T, held, lengths, H, D, page, heads, rot, interleaved):
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(T + H)
    B = len(held)
    caches, table, n = _pool(gen, dtype, held, T, page, H, D, heads)
    before = [c.clone() for c in caches]
    k, v = _rand(gen, dtype, B, T, H, D), _rand(gen, dtype, B, T, H, D)
    count = torch.tensor(lengths if lengths is not None else [T] * B, dtype=torch.int32, device=DEV)
    rotary = M.Rotary(M.rotary_frequencies(rot, device=DEV)[0], interleaved, 0.9) if rot else None
    M.paged_moda_append(k, v, *caches, table, n, None if lengths is None else count, rotary)
    assert M.last_launch_count() == 1
    at = n.long()[:, None] + torch.arange(T, device=DEV)
    want = turn(k.double(), at, rotary.inv_freq, interleaved, 0.9) if rot else k.double()
    tol = turn_bound(k.double(), want, rot, interleaved, 0.9, dtype) if rot else torch.zeros_like(want)
    for b in range(B):
        j = at[b, : int(count[b])]
        pages, slots = table[b, j // page].long(), j % page
        close(caches[0][pages, slots], want[b, : len(j)], tol[b, : len(j)], "keys")
        assert torch.equal(caches[1][pages, slots], v[b, : len(j)])
        for c, old in zip(caches, before):
            old[pages, slots] = c[pages, slots]
    for c, old in zip(caches, before):                                  # nothing else has been written
        assert torch.equal(c.view(torch.int16), old.view(torch.int16))
    assert M.device_status() == 0


# more tokens than warps run at once: two or four a warp, in steps
@pytest.mark.parametrize("dtype,T,held,lengths,H,D,page,heads,rot,interleaved", [
    (BF, 3001, [0, 5, 40, 17], [3001, 0, 2999, 1500], 6, 64, 64, True, 64, False),
    (HF, 5003, [3, 0], [5003, 4800], 5, 128, 24, False, 96, True),
])
def test_append_of_many_tokens(built_library, dtype, T, held, lengths, H, D, page, heads, rot, interleaved):
    test_append(built_library, dtype, T, held, lengths, H, D, page, heads, rot, interleaved)


@pytest.mark.parametrize("seed", range(8))
def test_drawn_calls(built_library, seed):
    """Calls of all kinds: sizes, divisions of the work, page sizes, layouts, depth rows of one or several positions, own rows, rotations.  Two calls in
    a row give the same bits (the second writes the same row again)."""
    import random

    import moda_b200 as M
    rng = random.Random(seed)
    for it in range(12):
        dtype, D, H, G = rng.choice([BF, HF]), rng.choice([64, 128]), rng.choice([1, 2, 3, 5, 8, 13]), rng.choice([1, 2, 3, 4, 7, 8, 9, 16])
        lens = rng.choice([
            lambda: [int(2 ** rng.uniform(0, 15))],
            lambda: [int(2 ** rng.uniform(0, 12)) - 1 for _ in range(rng.randint(2, 9))],
            lambda: [rng.randint(0, rng.choice([1, 5, 40, 200])) for _ in range(rng.randint(50, 400))],
            lambda: [int(2 ** rng.uniform(0, 11)) - 1 for _ in range(rng.randint(20, 60))],
            lambda: [rng.randint(3000, 12000)] + [rng.choice([0, 1, 2]) for _ in range(rng.randint(0, 20))],
        ])()
        page, room, own = rng.choice([1, 3, 8, 16, 17, 24, 32, 64, 100, 256]), rng.choice([1, 1, 500, 3000]), rng.random() < 0.5
        if len(lens) * (max(lens) + room) * H * D > 3e8:
            room = 1
            lens = lens[: max(1, int(3e8 / ((max(lens) + room) * H * D)))]
        B = len(lens)
        gen = torch.Generator(device=DEV).manual_seed(100 * seed + it)
        caches, table, n = _pool(gen, dtype, lens, room, page, H, D, rng.random() < 0.6)
        P, L, rot = rng.choice([0, 1, 1, 4]), rng.choice([1, 2, 7, 16, 33, 64]), rng.choice([0, 16, 64, D])
        depth, seen, kw = None, None, {}
        if P > 1:
            depth, seen = tuple(_rand(gen, dtype, B, P, L + 2, H, D)[:, :, :L] for _ in range(2)), [rng.randint(0, P) for _ in range(B)]
            kw["depth_positions"] = torch.tensor(seen, dtype=torch.int32, device=DEV)
        elif P == 1:
            depth = tuple(_rand(gen, dtype, B, L, H, D) for _ in range(2))
        if depth is not None:
            kw.update(cached_k=depth[0], cached_v=depth[1])
        if rot:
            kw["rotary"] = M.Rotary(M.rotary_frequencies(rot, device=DEV)[0], rng.random() < 0.5, rng.choice([1.0, 1.2]))
        if own:
            kw.update(k=_rand(gen, dtype, B, 1, H, D), v=_rand(gen, dtype, B, 1, H, D))
        q, scale = _rand(gen, dtype, B, G, H, D), rng.choice([D ** -0.5, 0.3, -0.1])
        o, lse = M.paged_moda_decode(q, *caches, table, n, **kw, scale=scale, moda_group_num=G, need_lse=True)
        again = M.paged_moda_decode(q, *caches, table, n, **kw, scale=scale, moda_group_num=G, need_lse=True)
        assert torch.equal(o, again[0]) and torch.equal(lse, again[1])
        turned = (kw["rotary"], n.long() - (0 if own else 1)) if rot else None
        _check_decode(o, lse, q, caches, table, [x + own for x in lens], scale, depth, turned, seen)
        assert M.device_status() == 0


def test_strides_scale_and_views(built_library):
    """Caches that are slices of something larger, queries and rows that are views, shared pages, and scales of either sign."""
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(9)
    B, H, G, D, page, L = 3, 2, 4, 64, 16, 3
    wide = torch.full((12, page, 2, H + 2, D + 8), float("nan"), device=DEV, dtype=BF)
    caches = [wide[:, :, i, 1 : H + 1, :D] for i in range(2)]
    lens = [70, 33, 16]
    table = torch.tensor([[0, 7, 3, 9, 1], [0, 7, 4, 11, 11], [0, 5, 5, 5, 5]], device=DEV, dtype=torch.int32)       # a common first page
    for c in caches:
        c.copy_(torch.randn(c.shape, generator=gen, device=DEV))
    wide_table = torch.zeros(B, 8, dtype=torch.int32, device=DEV)
    wide_table[:, 2:7] = table
    q = _rand(gen, BF, B, 2 * G, H + 1, D)[:, ::2, 1:]
    depth = [_rand(gen, BF, B, 5, 9, H, D).permute(0, 2, 1, 3, 4)[:, 1:3, :L] for _ in range(2)]
    n, seen = torch.tensor(lens, dtype=torch.int32, device=DEV), torch.tensor([2, 0, 1], dtype=torch.int32, device=DEV)
    for scale in (0.3, -0.2, 0.0, 4.0):
        o, lse = M.paged_moda_decode(q, *caches, wide_table[:, 2:7], n, cached_k=depth[0], cached_v=depth[1], depth_positions=seen,
                                     scale=scale, moda_group_num=G, need_lse=True)
        _check_decode(o, lse, q, caches, table, lens, scale, depth, seen=seen)
    odd = _rand(gen, BF, B, G, H, D + 1)[..., 1:]                       # not on a 16-byte boundary: copied
    o, lse = M.paged_moda_decode(odd, *caches, table, n, moda_group_num=G, need_lse=True)
    _check_decode(o, lse, odd, caches, table, lens, D ** -0.5)


def test_large_scores(built_library):
    """Scores of some hundreds, in growing and in falling order: the running maximum moves at every tile, or once."""
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(10)
    n, H, G, D, page = 700, 2, 2, 64, 32
    for order in (1, -1):
        caches, table, lens = _pool(gen, BF, [n], 0, page, H, D)
        q = torch.ones(1, G, H, D, device=DEV, dtype=BF)
        j = torch.arange(n, device=DEV)
        caches[0][table[0, j // page].long(), j % page] = (order * (j - n / 2) / 8).bfloat16()[:, None, None].expand(n, H, D)
        o, lse = M.paged_moda_decode(q, *caches, table, lens, moda_group_num=G, need_lse=True)
        _check_decode(o, lse, q, caches, table, [n], D ** -0.5)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_many_small_probabilities_beside_a_large_one(built_library, dtype):
    """60000 keys of e^-18 each: 9e-4 together, and each below 2^-25, fp16's smallest step.  Their values are all there is to the result."""
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(18)
    n, H, G, D, page = 60000, 1, 2, 64, 64
    caches, table, lens = _pool(gen, dtype, [n], 0, page, H, D)
    j = torch.arange(n, device=DEV)
    caches[0][table[0, j // page].long(), j % page] = torch.where(j == 31234, 0.0, -2.25)[:, None, None].expand(n, H, D).to(dtype)
    caches[1][table[0, j // page].long(), j % page] = torch.where(j == 31234, 0.0, 1.0)[:, None, None].expand(n, H, D).to(dtype)
    q = torch.ones(1, G, H, D, device=DEV, dtype=dtype)
    o, lse = M.paged_moda_decode(q, *caches, table, lens, moda_group_num=G, need_lse=True)
    assert abs(o[0, 0, 0, 0].item() - 9.1e-4) < 1e-5
    _check_decode(o, lse, q, caches, table, [n], D ** -0.5)


def test_turned_queries_beyond_fp16(built_library):
    """Pairs of 60000 turn to up to 84853, which fp16 does not hold; the score of small keys is an ordinary number."""
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(19)
    lens, H, G, D, page = [50, 7, 300], 2, 2, 64, 16
    caches, table, n = _pool(gen, HF, lens, 1, page, H, D)
    caches[0].mul_(1e-5)
    rotary = M.Rotary(M.rotary_frequencies(D, device=DEV)[0])
    q = torch.where(torch.rand(3, G, H, D, generator=gen, device=DEV) < 0.5, -60000.0, 60000.0).half()
    o, lse = M.paged_moda_decode(q, *caches, table, n, rotary=rotary, moda_group_num=G, need_lse=True)
    _check_decode(o, lse, q, caches, table, lens, D ** -0.5, None, (rotary, n.long() - 1))


def test_nan_stays_where_it_belongs(built_library):
    """A NaN key of one sequence's head spoils that head's result and no other."""
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(11)
    lens = [40, 40]
    caches, table, n = _pool(gen, HF, lens, 0, 16, 2, 64)
    caches[0][table[0, 1].long(), 3, 1] = float("nan")
    q = _rand(gen, HF, 2, 2, 2, 64)
    o, lse = M.paged_moda_decode(q, *caches, table, n, moda_group_num=2, need_lse=True)
    assert o[0, :, 1].isnan().all() and lse[0, :, 1].isnan().all()
    assert not o[0, :, 0].isnan().any() and not o[1].isnan().any() and not lse[1].isnan().any()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("turned", [False, True])
def test_infinite_keys_and_values(built_library, dtype, turned):
    """An infinite element of a key makes its score infinite, of either sign: +inf gives NaN, as the quotient inf / inf does, -inf leaves the
    key out.  An infinite value makes its element of the result infinite.  No other sequence, head or element notices."""
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(20)
    lens, H, G, D, page = [40, 40, 40, 40], 2, 2, 64, 16
    caches, table, n = _pool(gen, dtype, lens, 0, page, H, D)
    q = _rand(gen, dtype, 4, G, H, D).abs() + 0.25
    rotary = M.Rotary(M.rotary_frequencies(16, device=DEV)[0]) if turned else None      # the elements concerned do not turn
    at = table[:, 1].long()
    caches[0][at[0], 3, 1, 40] = float("inf")
    caches[0][at[1], 3, 1, 40] = float("-inf")
    caches[1][at[2], 3, 1, 40] = float("inf")
    o, lse = M.paged_moda_decode(q, *caches, table, n, rotary=rotary, moda_group_num=G, need_lse=True)
    assert o[0, :, 1].isnan().all()
    assert (o[2, :, 1, 40] == float("inf")).all()
    clean = [c.clone() for c in caches]
    clean[0][at[0], 3, 1, 40] = clean[1][at[2], 3, 1, 40] = 0
    clean[0][at[1], 3, 1, 40] = -60000.0                    # far enough below: its probability is 0 too
    want, want_lse = M.paged_moda_decode(q, *clean, table, n, rotary=rotary, moda_group_num=G, need_lse=True)
    same = torch.ones_like(o, dtype=torch.bool)
    same[0, :, 1] = same[2, :, 1, 40] = False
    assert torch.equal(o[same], want[same])
    assert torch.equal(lse[1:], want_lse[1:]) and torch.equal(lse[0, :, 0], want_lse[0, :, 0])


def test_bad_tables_and_lengths_are_left_out_and_recorded(built_library):
    """Page numbers outside the pool: the kernels look at each before they use it.  Lengths outside the table: bounded by it."""
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(12)
    H, G, D, page = 2, 2, 64, 16
    lens = [60, 50]
    caches, table, n = _pool(gen, BF, lens, 4, page, H, D)
    q = _rand(gen, BF, 2, G, H, D)
    pages = caches[0].shape[0]
    for bad in (-1, pages, 2 ** 31 - 1, -2 ** 31):
        broken = table.clone()
        broken[0, 1] = bad
        o, lse = M.paged_moda_decode(q, *caches, broken, n, moda_group_num=G, need_lse=True)
        assert M.device_status() == (2 << 8 | 1) and M.device_status() == 0
        keep = [j for j in range(60) if j // page != 1]
        keys, values = (rows_of(c, table[0], 60)[keep].double() for c in caches)
        want = attend(q[0].double(), keys, values, D ** -0.5)
        tol = attend_bounds(*want, D, BF, False)
        close(o[0], want[0], tol[0], "o"), close(lse[0], want[1], tol[1], "lse")
        _check_decode(o[1:], lse[1:], q[1:], caches, table[1:], lens[1:], D ** -0.5)
        before = [c.clone() for c in caches]
        M.paged_moda_append(_rand(gen, BF, 2, 4, H, D), _rand(gen, BF, 2, 4, H, D), *caches, broken, torch.tensor([16, 50], dtype=torch.int32, device=DEV),
                            torch.tensor([4, 0], dtype=torch.int32, device=DEV))
        assert M.device_status() == (2 << 8 | 1)
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(caches, before))
    depth = [_rand(gen, BF, 2, 3, 2, H, D) for _ in range(2)]
    for bad, seen in ((4, 3), (-1, 0)):
        positions = torch.tensor([bad, 2], dtype=torch.int32, device=DEV)
        o, lse = M.paged_moda_decode(q, *caches, table, n, cached_k=depth[0], cached_v=depth[1], depth_positions=positions, moda_group_num=G, need_lse=True)
        assert M.device_status() == (2 << 8 | 2)
        _check_decode(o, lse, q, caches, table, lens, D ** -0.5, depth, seen=[seen, 2])
    room = table.shape[1] * page
    full, ftable, _ = _pool(gen, BF, [room, room], 0, page, H, D)
    for bad, seen in (([-5, room], [0, room]), ([room + 1, 3], [room, 3]), ([2 ** 31 - 1, -2 ** 31], [room, 0])):
        n = torch.tensor(bad, dtype=torch.int32, device=DEV)
        o, lse = M.paged_moda_decode(q, *full, ftable, n, moda_group_num=G, need_lse=True)
        assert M.device_status() == (2 << 8 | 2)
        _check_decode(o, lse, q, full, ftable, seen, D ** -0.5)
        before = [c.clone() for c in full]
        M.paged_moda_append(_rand(gen, BF, 2, 1, H, D), _rand(gen, BF, 2, 1, H, D), *full, ftable, n, torch.tensor([1, 0 if bad[1] == 3 else 1], dtype=torch.int32, device=DEV))
        assert M.device_status() == (2 << 8 | 2)
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(full, before))


@pytest.mark.parametrize("what", ["no room", "bad page", "negative length"])
def test_a_row_without_a_place(built_library, what):
    """The token's own row has nowhere to go: it is left out of the result too, nothing is written, and the other sequences go on."""
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(21)
    H, G, D, page = 2, 9, 64, 16
    lens = [48, 33, 20]
    caches, table, n = _pool(gen, BF, lens, 0, page, H, D)
    table = table.clone()
    if what == "bad page":
        lens = [33, 33, 20]
        table[0, 2] = -1
    n = torch.tensor([-7 if what == "negative length" else lens[0], *lens[1:]], dtype=torch.int32, device=DEV)
    held = {"no room": 48, "bad page": 32, "negative length": 0}[what]
    before = [c.clone() for c in caches]
    q, k, v = _rand(gen, BF, 3, G, H, D), _rand(gen, BF, 3, 1, H, D), _rand(gen, BF, 3, 1, H, D)
    record = [torch.full((3, 1, H, D), 7.0, device=DEV, dtype=BF) for _ in range(2)]
    o, lse = M.paged_moda_decode(q, *caches, table, n, k, v, moda_group_num=G, need_lse=True, record_k=record[0], record_v=record[1])
    assert M.device_status() == (2 << 8 | (1 if what == "bad page" else 2))
    _check_decode(o, lse, q, caches, table, [held, 34, 21], D ** -0.5)
    assert (record[0][0] == 7).all() and (record[1][0] == 7).all() and torch.equal(record[0][1:], k[1:]) and torch.equal(record[1][1:], v[1:])
    for c, old, new in zip(caches, before, (k, v)):
        for b in (1, 2):
            old[table[b, lens[b] // page].long(), lens[b] % page] = new[b, 0]
        assert torch.equal(c.view(torch.int16), old.view(torch.int16))


def test_offsets_past_32_bits(built_library):
    """A pool of more than 2^32 bytes: the sequences' pages are its first and its last ones."""
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(13)
    H, G, D, page = 8, 4, 128, 64
    pages = (2 ** 31 + 2 ** 24) // (H * D * page)
    caches = [torch.empty(pages, H, page, D, device=DEV, dtype=BF).transpose(1, 2) for _ in range(2)]
    table = torch.tensor([[pages - 1, 0, pages - 2, pages - 3]], device=DEV, dtype=torch.int32)
    for c in caches:
        c[table[0].long()] = torch.randn(4, page, H, D, generator=gen, device=DEV).to(BF)
    q, k, v = _rand(gen, BF, 1, G, H, D), _rand(gen, BF, 1, 1, H, D), _rand(gen, BF, 1, 1, H, D)
    n = torch.tensor([200], dtype=torch.int32, device=DEV)
    o, lse = M.paged_moda_decode(q, *caches, table, n, k, v, moda_group_num=G, need_lse=True)
    _check_decode(o, lse, q, caches, table, [201], D ** -0.5)
    assert torch.equal(caches[1][pages - 3, 200 - 192], v[0, 0])
    M.paged_moda_append(k, v, *caches, table, torch.tensor([5], dtype=torch.int32, device=DEV))
    assert torch.equal(caches[0][pages - 1, 5], k[0, 0])


def test_refusals_on_the_gpu(built_library):
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(14)
    caches, table, n = _pool(gen, BF, [5], 3, 8, 2, 64)
    q, k = _rand(gen, BF, 1, 1, 2, 64), _rand(gen, BF, 1, 1, 2, 64)
    with pytest.raises(RuntimeError, match="does not train"):
        M.paged_moda_decode(q.clone().requires_grad_(), *caches, table, n)
    with pytest.raises(RuntimeError, match="does not train"):
        M.paged_moda_append(k.clone().requires_grad_(), k, *caches, table, n)
    with torch.no_grad():
        M.paged_moda_decode(q.clone().requires_grad_(), *caches, table, n)
    with pytest.raises(AssertionError, match="dtype and device"):
        M.paged_moda_decode(q.half(), *caches, table, n)
    with pytest.raises(AssertionError, match="one device"):
        M.paged_moda_decode(q, *caches, table.cpu(), n)
    with pytest.raises(TypeError, match="bf16/fp16"):
        M.paged_moda_append(k.float(), k.float(), caches[0].float(), caches[1].float(), table, n)
    with pytest.raises(M.ModaLibraryError) as e:
        M.paged_moda_append(k[:, :0], k[:, :0], *caches, table, n)
    assert e.value.status == 2


@pytest.mark.parametrize("lens", [[900, 0, 33], [9000, 5, 20]])       # short enough for clusters; divided evenly
def test_captured_steps_follow_the_lengths(built_library, lens):
    """A decoding step is captured once and replayed while the sequences grow, behind a copy and behind another stream's work; two
    captured graphs and an eager call share nothing."""
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(15)
    H, G, D, page, B = 2, 4, 128, 16, 3
    caches, table, n = _pool(gen, BF, lens, 12, page, H, D)
    rotary = M.Rotary(M.rotary_frequencies(D, device=DEV)[0])
    q, k, v = _rand(gen, BF, B, G, H, D), _rand(gen, BF, B, 1, H, D), _rand(gen, BF, B, 1, H, D)

    other, given, also = torch.cuda.Stream(), q.clone(), torch.zeros(1 << 16, device=DEV)

    def step():
        here = torch.cuda.current_stream()
        other.wait_stream(here)
        with torch.cuda.stream(other):
            also.add_(1)
        q.copy_(given)                                                   # a copy, not a kernel, is what comes before
        here.wait_stream(other)
        r = M.paged_moda_decode(q, *caches, table, n, k, v, rotary=rotary, moda_group_num=G, need_lse=True)
        n.add_(1)
        return r

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graphs, outs = [], []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(step())
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(side)
    assert n.tolist() == [x + 1 for x in lens]
    for i in range(5):
        for x in (given, k, v):
            x.copy_(_rand(gen, BF, *x.shape))
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        now = [x + 2 + i for x in lens]
        assert n.tolist() == now
        _check_decode(*outs[i % 2], q, caches, table, now, D ** -0.5, None, (rotary, n.long() - 1))
    assert M.device_status() == 0


@pytest.mark.parametrize("dtype,lens,H,G,D,P,L,page", [
    (BF, [(7 * i) % 100 for i in range(101)], 3, 4, 128, 1, 8, 16),
    (HF, [i % 3 for i in range(230)], 2, 9, 64, 1, 3, 8),
    (HF, [(11 * i) % 64 for i in range(1500)], 1, 2, 64, 0, 0, 64),
    (BF, [i % 50 for i in range(150)], 4, 2, 128, 2, 5, 32),
    (BF, [(5 * i) % 90 for i in range(120)], 4, 3, 64, 4, 64, 64),        # short but for its depth rows
])
def test_more_short_units_than_ctas(built_library, dtype, lens, H, G, D, P, L, page):
    """Where the table lets no sequence be long and there are more units than CTAs, warps take whole units: nothing is joined."""
    import moda_b200 as M
    from moda_b200 import _cabi
    gen = torch.Generator(device=DEV).manual_seed(18)
    B = len(lens)
    caches, table, n = _pool(gen, dtype, lens, 3, page, H, D)
    rotary = M.Rotary(M.rotary_frequencies(D, device=DEV)[0])
    q, k, v = _rand(gen, dtype, B, G, H, D), _rand(gen, dtype, B, 1, H, D), _rand(gen, dtype, B, 1, H, D)
    depth, seen, kw = None, None, {}
    if P > 1:
        depth, seen = [_rand(gen, dtype, B, P, L, H, D) for _ in range(2)], [i % (P + 1) for i in range(B)]
        kw = dict(cached_k=depth[0], cached_v=depth[1], depth_positions=torch.tensor(seen, dtype=torch.int32, device=DEV))
    elif P == 1:
        depth = [_rand(gen, dtype, B, L, H, D) for _ in range(2)]
        kw = dict(cached_k=depth[0], cached_v=depth[1])
    _cabi.profile_begin()
    o, lse = M.paged_moda_decode(q, *caches, table, n, moda_group_num=G, need_lse=True, **kw)
    assert "paged_decode" in (ran := _cabi.profile_end()) and "paged_join" not in ran
    _check_decode(o, lse, q, caches, table, lens, D ** -0.5, depth, seen=seen)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = M.paged_moda_decode(q, *caches, table, n, k, v, rotary=rotary, moda_group_num=G, need_lse=True, **kw)
        n.add_(1)
    for i in range(2):
        graph.replay()
        now = [x + 1 + i for x in lens]
        _check_decode(o, lse, q, caches, table, now, D ** -0.5, depth, (rotary, n.long() - 1), seen)
    assert M.device_status() == 0

    # a page of one sequence outside the pool, lengths of two outside the table
    at = [i for i in range(B) if now[i] > 0]
    broken, bad = table.clone(), n.clone()
    broken[at[1], 0] = -1
    o, lse = M.paged_moda_decode(q, *caches, broken, n, moda_group_num=G, need_lse=True, **kw)
    assert M.device_status() == (2 << 8 | 1)
    room = table.shape[1] * page
    bad[at[0]], bad[at[-1]] = -3, room + 1
    o2, lse2 = M.paged_moda_decode(q, *caches, table, bad, moda_group_num=G, need_lse=True, **kw)
    assert M.device_status() == (2 << 8 | 2)
    want, want_lse = M.paged_moda_decode(q, *caches, table, n, moda_group_num=G, need_lse=True, **kw)
    for x, y, but in ((o, want, [at[1]]), (lse, want_lse, [at[1]]), (o2, want, [at[0], at[-1]]), (lse2, want_lse, [at[0], at[-1]])):
        others = [i for i in range(B) if i not in but]
        assert torch.equal(x[others], y[others])


def test_calls_on_several_streams_at_once(built_library):
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(16)
    H, G, D, page = 4, 4, 128, 64
    sets = []
    for lens in ([6000, 10], [3000, 5000, 1], [200, 90], [300]):         # divided evenly, and over clusters
        caches, table, n = _pool(gen, BF, lens, 0, page, H, D)
        sets.append((lens, caches, table, n, _rand(gen, BF, len(lens), G, H, D)))
    want = [M.paged_moda_decode(q, *caches, table, n, moda_group_num=G, need_lse=True) for _, caches, table, n, q in sets]
    for (lens, caches, table, n, q), (o, lse) in zip(sets, want):
        _check_decode(o, lse, q, caches, table, lens, D ** -0.5)
    streams, got = [torch.cuda.Stream() for _ in sets], [[] for _ in sets]
    for _ in range(20):
        for i, (_, caches, table, n, q) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append(M.paged_moda_decode(q, *caches, table, n, moda_group_num=G, need_lse=True))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        assert all(torch.equal(w[0], g[0]) and torch.equal(w[1], g[1]) for g in gs)


def test_writes_are_noticed_by_autograd(built_library):
    import moda_b200 as M
    H, G, D = 2, 2, 64
    cache = M.PagedKVCache(4, 16, H, D, BF, "cuda")
    cache.k.zero_()
    cache.v.zero_()
    table = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    n = torch.tensor([5], dtype=torch.int32, device="cuda")
    q, k, record = (torch.randn(1, t, H, D, device="cuda").to(BF) for t in (G, 1, 1))
    w = torch.ones(D, device="cuda", dtype=BF, requires_grad=True)

    def saved(x):                            # the gradient of w reads x
        return (x * w).sum()

    y = [saved(x) for x in (cache.k, cache.v, record)]
    cache.decode(q, table, n, moda_group_num=G)                           # reads only
    for x in y:
        x.backward(retain_graph=True)
    for write in (lambda: cache.append(k, k, table, n), lambda: cache.decode(q, table, n, k, k, moda_group_num=G)):
        y = [saved(x) for x in (cache.k, cache.v)]
        write()
        for x in y:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                x.backward()
    y = saved(record)
    M.paged_moda_decode(q, cache.k, cache.v, table, n, k, k, moda_group_num=G, record_k=record, record_v=torch.empty_like(record))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():             # these tensors have no version
        cache = M.PagedKVCache(4, 16, H, D, BF, "cuda")
        cache.append(k, k, table, n)
        cache.decode(q, table, n, k, k, moda_group_num=G)


@pytest.mark.parametrize("chunk_visible,G", [(False, 2), (False, 1), (True, 4)])
def test_generating_with_a_stack_of_layers(built_library, chunk_visible, G):
    """A prompt through the operators and its K/V into the caches, then tokens one by one: the attention of each layer at each new
    position is what the operator over the whole sequence gives there."""
    import moda_b200 as M
    from oracle import moda_oracle as mo
    gen = torch.Generator(device=DEV).manual_seed(17)
    B, T0, T, H, D, N, page = 2, 37, 45, 2, 64, 4, 16
    rotary = M.Rotary(M.rotary_frequencies(D, device=DEV)[0])
    C = 64 // G
    layers = [tuple(_rand(gen, BF, B, T * r, H, D) for r in (G, 1, 1)) for _ in range(N)]
    turned = [(*M.rotary_embedding(q, k, rotary, moda_group_num=G), v) for q, k, v in layers]
    pages = [M.PagedKVCache(B * 3, page, H, D, BF, DEV) for _ in range(N)]
    table = torch.arange(B * 3, device=DEV, dtype=torch.int32).view(B, 3)
    n = torch.zeros(B, dtype=torch.int32, device=DEV)
    for cache, (_, k, v) in zip(pages, layers):
        cache.append(k[:, :T0], v[:, :T0], table, n, rotary=rotary)
    n += T0
    for t in range(T0, T):
        first = t // C * C if chunk_visible else t                      # the positions whose depth rows the token sees
        depth = M.DepthKVCache(B, t + 1 - first, N - 1, H, D, BF, DEV)
        for i, (cache, (q, k, v)) in enumerate(zip(pages, layers)):
            row = (q[:, t * G : (t + 1) * G], table, n, k[:, t : t + 1], v[:, t : t + 1])
            if chunk_visible:
                seen = torch.full((B,), t + 1 - first, dtype=torch.int32, device=DEV)
                o, lse = cache.decode(*row, depth=depth, depth_positions=seen, moda_group_num=G, rotary=rotary, need_lse=True)
                if i + 1 < N:
                    depth.append(turned[i][1][:, first : t + 1], turned[i][2][:, first : t + 1])
            else:
                o, lse = cache.decode(*row, depth=depth, record=i + 1 < N, moda_group_num=G, rotary=rotary, need_lse=True)
            assert depth.L == min(i + 1, N - 1)
            qt, kt, vt = (x[:, : (t + 1) * r].float().cpu() for x, r in zip(turned[i], (G, 1, 1)))
            kd, vd = (torch.stack([x[j][:, : t + 1] for x in turned[:i]], 2).flatten(1, 2).float().cpu() if i else None for j in (1, 2))
            ref_o, ref_lse = mo.moda_attention_ref(qt, kt, vt, kd, vd, None, G, mo.MODE_CHUNK_VISIBLE if chunk_visible else mo.MODE_CAUSAL, C)
            # The oracle takes q rounded to bf16, the step turns it without rounding: a score is off by 2^-9 of up to
            # scale * sum |q k| (about 8 here, terms of either sign), and o by a few 2^-8 of values of about 1.
            assert (o.float().cpu() - ref_o[:, -G:]).abs().max() <= 2e-2
            assert (lse.cpu() - ref_lse[:, -G:]).abs().max() <= 2e-2
        n += 1
    for cache, (_, k, v) in zip(pages, turned):                         # and the caches hold every row
        for b in range(B):
            assert torch.equal(rows_of(cache.k, table[b], T), k[b]) and torch.equal(rows_of(cache.v, table[b], T), v[b])
    assert M.device_status() == 0


def test_any_stride_where_there_is_one_row(built_library):
    """Pages of one row, one depth layer (of one position and of several), one head and one sequence, whose strides are not multiples of 8."""
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(22)
    G, D = 3, 64

    def odd(x, dim):                                                     # the same memory, stride 65 where the extent is 1
        assert x.shape[dim] == 1
        stride = list(x.stride())
        stride[dim] = 65
        return x.as_strided(x.shape, stride)

    for B, H, page, L, P in ((2, 2, 1, 1, 1), (3, 2, 1, 1, 2), (1, 1, 16, 1, 1), (2, 1, 24, 1, 3), (1, 2, 1, 5, 1)):
        lens = [19, 1, 16][:B]
        caches, table, n = _pool(gen, BF, lens, 2, page, H, D, heads=False)
        q, k, v = _rand(gen, BF, B, G, H, D), _rand(gen, BF, B, 1, H, D), _rand(gen, BF, B, 1, H, D)
        depth = [_rand(gen, BF, B, P, L, H, D) for _ in range(2)]
        seen = list(range(P, P - B, -1)) if P > 1 else None
        given = [c for c in caches]
        if page == 1:
            given = [odd(c, 1) for c in given]
        if H == 1:
            given, q, k, v = [odd(c, 2) for c in given], odd(q, 2), odd(k, 2), odd(v, 2)
        if B == 1:
            q = odd(q, 0)
        rows = [x if P > 1 else x[:, 0] for x in depth]
        if L == 1:
            rows = [odd(x, x.dim() - 3) for x in rows]
        kw = dict(depth_positions=torch.tensor(seen, dtype=torch.int32, device=DEV)) if P > 1 else {}
        o, lse = M.paged_moda_decode(q, *given, table, n, odd(k, 1), odd(v, 1), *rows, **kw, moda_group_num=G, need_lse=True)
        _check_decode(o, lse, q, caches, table, [x + 1 for x in lens], D ** -0.5, depth if P > 1 else rows, seen=seen)
        n += 1
        M.paged_moda_append(odd(k, 1), odd(v, 1), *given, table, n)
        for b, at in enumerate(lens):
            assert torch.equal(caches[0][table[b, (at + 1) // page].long(), (at + 1) % page], k[b, 0])
    assert M.device_status() == 0


@pytest.mark.parametrize("dtype,B,G,D,page,pages_each,long", [
    (BF, 3, 9, 64, 16, 20, 300),            # a unit to a cluster
    (HF, 4, 2, 128, 16, 2, 32),             # to a CTA
    (HF, 8, 4, 128, 16, 1200, 9600),        # divided evenly
    (BF, 900, 3, 64, 16, 3, 48),            # whole units to warps
    (HF, 700, 2, 128, 16, 40, 60),          # divided evenly, short units to warps
])
@pytest.mark.parametrize("turned", [False, True])
def test_the_next_layer_sees_a_row_without_a_place(built_library, dtype, B, G, D, page, pages_each, long, turned):
    """Two layers over a depth cache that holds NaN: sequences whose row the table has no room for, whose page is none of the pool's, or whose length is
    negative.  The first layer leaves the row out; it is the second layer's depth row all the same, turned at the position that the query takes."""
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(23)
    H = 2
    room = pages_each * page
    table = torch.randperm(B * pages_each, generator=gen, device=DEV).view(B, pages_each).int()
    lens = [min(long, room - 1) - (7 * b) % 30 for b in range(B)]
    broken = {0: "no room", B // 2: "bad page", B - 1: "negative"}
    lens[0], lens[B // 2] = room, 33 if room > 33 else 17
    table[B // 2, lens[B // 2] // page] = -1 if B % 2 else B * pages_each
    held = [0 if broken.get(b) == "negative" else x for b, x in enumerate(lens)]
    n = torch.tensor([-5 if broken.get(b) == "negative" else x for b, x in enumerate(lens)], dtype=torch.int32, device=DEV)
    at = torch.tensor(held, device=DEV)
    rotary = M.Rotary(M.rotary_frequencies(D, device=DEV)[0], True, 1.1) if turned else None
    layers = [M.PagedKVCache(B * pages_each, page, H, D, dtype, DEV) for _ in range(2)]
    depth = M.DepthKVCache(B, 1, 3, H, D, dtype, DEV)
    for x in (depth.k, depth.v):
        x.fill_(float("nan"))
    rows = []
    for i, layer in enumerate(layers):
        for x in (layer.k, layer.v):
            x.copy_(torch.randn(x.shape, generator=gen, device=DEV))
        q, k, v = _rand(gen, dtype, B, G, H, D), _rand(gen, dtype, B, 1, H, D), _rand(gen, dtype, B, 1, H, D)
        before = [layer.k.clone(), layer.v.clone()]
        o, lse = layer.decode(q, table, n, k, v, depth=depth, record=True, moda_group_num=G, rotary=rotary, need_lse=True)
        assert M.device_status() in ((2 << 8 | 1), (2 << 8 | 2)) and M.device_status() == 0 and depth.L == i + 1
        for b, why in broken.items():
            keys, values = (rows_of(c, table[b].clamp(0, B * pages_each - 1), held[b]).double() for c in (layer.k, layer.v))
            if why == "bad page":
                first = held[b] // page * page
                keys, values = keys[:first], values[:first]
            if i:
                keys, values = torch.cat([keys, rows[0][b].double()]), torch.cat([values, rows[1][b].double()])
            q64 = turn(q[b : b + 1].double(), at[b : b + 1, None], rotary.inv_freq, True, 1.1)[0] if turned else q[b].double()
            want = attend(q64, keys, values, D ** -0.5)
            tol = attend_bounds(*want, D, dtype, turned)
            close(o[b], want[0], tol[0], why), close(lse[b], want[1], tol[1], why)
        others = [b for b in range(B) if b not in broken][:40]
        _check_decode(o[others], lse[others], q[others], (layer.k, layer.v), table[others], [lens[b] + 1 for b in others], D ** -0.5,
                      [x[others] for x in rows] if i else None, (rotary, at[others]) if turned else None)
        rows = [x.view(B, 3, H, D)[:, i : i + 1].clone() for x in (depth.k, depth.v)]
        want_k = turn(k.double(), at[:, None], rotary.inv_freq, True, 1.1) if turned else k.double()
        close(rows[0], want_k, turn_bound(k.double(), want_k, D, True, 1.1, dtype) if turned else torch.zeros_like(want_k), "recorded keys")
        assert torch.equal(rows[1], v)
        ok = torch.tensor([b for b in range(B) if b not in broken], dtype=torch.long, device=DEV)
        pages, slots = table[ok, at[ok] // page].long(), at[ok] % page
        for c, old, new in zip((layer.k, layer.v), before, rows):        # nothing else has been written
            old[pages, slots] = new[ok, 0]
            assert torch.equal(c, old)
    if not turned:                                                       # an infinite value of a row that is left out counts nowhere
        v[:] = float("inf")
        want = layer.decode(q, table, n, k, torch.zeros_like(v), depth=depth, moda_group_num=G)[list(broken)]
        assert torch.equal(layer.decode(q, table, n, k, v, depth=depth, moda_group_num=G)[list(broken)], want)
        assert M.device_status() != 0


@pytest.mark.parametrize("which", ["record_k", "record_v", "both", "views of a leaf"])
def test_records_that_require_gradients_are_refused(built_library, which):
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(24)
    caches, table, n = _pool(gen, BF, [5], 3, 8, 2, 64, fill=0.0)
    q, k = _rand(gen, BF, 1, 1, 2, 64), _rand(gen, BF, 1, 1, 2, 64)
    before = [c.clone() for c in caches]
    leaf = torch.zeros(2, 1, 1, 2, 64, device=DEV, dtype=BF)
    rk, rv = (leaf.requires_grad_()[0], leaf[1]) if which == "views of a leaf" else (leaf[0].clone(), leaf[1].clone())
    if which != "views of a leaf":
        rk.requires_grad_(which != "record_v"), rv.requires_grad_(which != "record_k")
    with pytest.raises(RuntimeError, match="does not train"):
        M.paged_moda_decode(q, *caches, table, n, k, k, record_k=rk, record_v=rv)
    assert not rk.any() and not rv.any() and all(torch.equal(a, b) for a, b in zip(caches, before))
    with torch.no_grad():
        M.paged_moda_decode(q, *caches, table, n, k, k, record_k=rk, record_v=rv)
    assert torch.equal(rk, k) and torch.equal(rv, k)


@pytest.mark.parametrize("H,D,T", [(2, 64, 3), (20, 128, 5), (1, 64, 40)])
@pytest.mark.parametrize("bad", [-1, -(2 ** 31), "T + 1", 2 ** 31 - 1])
def test_append_of_more_tokens_than_there_are(built_library, H, D, T, bad):
    """A length of the call that is negative or more than T is recorded; what there is is written, and no more."""
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(25)
    bad = T + 1 if bad == "T + 1" else bad
    held, page = [7, 0, 16], 8
    caches, table, n = _pool(gen, BF, held, T + 3, page, H, D)
    before = [c.clone() for c in caches]
    k, v = _rand(gen, BF, 3, T, H, D), _rand(gen, BF, 3, T, H, D)
    M.paged_moda_append(k, v, *caches, table, n, torch.tensor([T, 0, 1], dtype=torch.int32, device=DEV))
    assert M.device_status() == 0
    M.paged_moda_append(k, v, *caches, table, n, torch.tensor([T, bad, 1], dtype=torch.int32, device=DEV))
    assert M.device_status() == (2 << 8 | 2) and M.device_status() == 0
    for b, count in enumerate([T, 0 if bad < 0 else T, 1]):
        at = held[b] + torch.arange(count, device=DEV)
        for old, x in zip(before, (k, v)):
            old[table[b, at // page].long(), at % page] = x[b, :count]
    assert all(torch.equal(c.view(torch.int16), old.view(torch.int16)) for c, old in zip(caches, before))


def test_status_waits_for_streams_of_any_kind(built_library):
    """A stream that does not wait for the default one, with work in front of the call that leaves something out."""
    import moda_b200 as M
    gen = torch.Generator(device=DEV).manual_seed(26)
    caches, table, n = _pool(gen, BF, [5], 3, 8, 2, 64)
    k = _rand(gen, BF, 1, 1, 2, 64)
    broken = table.clone()
    broken[0, 0] = -1
    a = torch.randn(8192, 8192, device=DEV, dtype=BF)
    side = torch.cuda.Stream()
    for t, times in ((table, 1), (broken, 60)):          # a first launch may wait for the device by itself
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(times):
                b = a @ a
            M.paged_moda_append(k, k, *caches, t, n)
        assert M.device_status() == (0 if t is table else 2 << 8 | 1) and M.device_status() == 0
    assert side.query() and b.shape == a.shape
