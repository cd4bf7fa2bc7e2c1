"""The paged 8-bit cache: plan, writes and attention, each against its definition in 64 bits (tests/_kv_ref.py), alone and as a
serving loop uses them."""
import math

import numpy as np
import pytest
import torch

import torch_mlu_amd as tm
from tests import _kv_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, F8, I8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.int8


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


# ---- plan -------------------------------------------------------------------------------------------------------------
def _plan_case(cached, new, width, page, max_tokens, capacity, count, seed=0):
    r = np.random.RandomState(seed)
    table = r.randint(0, 1000, (len(cached), width)).astype(np.int32)
    free = r.permutation(capacity).astype(np.int32) + 1000
    want = ref.plan(cached, new, table, free, count, page, max_tokens)
    t, f = ints(table), ints(free)
    got = tm.paged_plan(ints(cached), ints(new), t, f, ints([count]), page_size=page, max_tokens=max_tokens)
    assert torch.equal(f.cpu(), torch.from_numpy(free))
    assert np.array_equal(t.cpu().numpy(), want["table"])
    for n in got._fields:
        assert np.array_equal(getattr(got, n).cpu().numpy(), want[n]), n
    assert (got.cu_seqlens.dtype, got.slots.dtype, got.admitted.dtype) == (torch.int32, torch.int64, torch.bool)
    return want


@pytest.mark.parametrize("cached,new,width,page,tokens,capacity,count", [
    ([0], [1], 4, 64, 1, 3, 3),                                  # the first token of a request takes a page
    ([64], [1], 4, 64, 1, 3, 3), ([63], [1], 4, 64, 1, 3, 3),    # at a page's border, just before it
    ([5, 0, 130], [0, 0, 0], 4, 64, 0, 3, 3),                    # nothing new
    ([5, 0, 130], [0, 0, 0], 4, 64, 7, 3, 3),                    # ... in a padded step
    ([3, 200, 0, 64], [1, 300, 129, 1], 16, 32, 500, 40, 40),    # prompts and decodes, padded
    ([3, 200, 0, 64], [1, 300, 129, 1], 16, 32, 431, 13, 13),    # a page short: the prompt in the middle
    ([0, 0, 0, 0, 31], [33, 33, 33, 33, 1], 2, 32, 200, 50, 5),  # the later ones go without, one that needs no page is admitted
    ([0, 0, 0], [33, 0, 33], 2, 32, 66, 50, 0),                  # nothing free
    ([0, 60], [100, 5], 2, 32, 120, 9, 9),                       # a row of the table is full: not admitted, takes no page
    ([0, 0, 5], [10, 10, 10], 4, 32, 25, 9, 9),                  # beyond the step's rows
    ([-5, 10], [-3, 4], 4, 32, 10, 9, 9),                        # below 0 counts as 0
    ([7, 9], [3, 70], 4, 5, 80, 30, 30),                         # a page size that is no power of two
    ([0, 1], [4, 4], 4, 32, 8, 3, 99), ([0, 1], [4, 4], 4, 32, 8, 3, -2),   # a count that the list does not have
    ([0], [1], 0, 32, 4, 3, 3),                                  # a table without columns
    ([2 ** 31 - 1, 4], [2 ** 31 - 1, 1], 4, 32, 9, 3, 3),        # sums beyond 32 bits
])
def test_plan(cached, new, width, page, tokens, capacity, count):
    _plan_case(cached, new, width, page, tokens, capacity, count)


@pytest.mark.parametrize("B,seed", [(1, 1), (63, 2), (64, 3), (65, 4), (1000, 5), (1024, 6), (1025, 7), (3000, 8), (8192, 9)])
def test_plan_random(B, seed):
    r = np.random.RandomState(seed)
    cached, new = r.randint(0, 300, B), np.where(r.rand(B) < 0.1, r.randint(0, 200, B), r.randint(0, 2, B))
    total = int(new.sum())
    for short in (0, 1):
        w = _plan_case(cached.tolist(), new.tolist(), 17, 32, max(0, total + 13 - 20 * short), 5 * B + 200, B // 8 + 1 if short else 5 * B + 200, seed)
        assert w["admitted"].all() == (not short)


def test_plan_of_no_requests():
    got = tm.paged_plan(ints([]), ints([]), torch.zeros(0, 4, dtype=torch.int32, device=DEV), ints([3]), ints([1]), page_size=32, max_tokens=5)
    assert got.cu_seqlens.tolist() == [0] and got.slots.tolist() == [-1] * 5 and got.positions.tolist() == [0] * 5 and got.free_count.tolist() == [1]


def test_plan_table_that_is_a_slice_and_a_negative_page():
    wide = torch.full((3, 20), -7, dtype=torch.int32, device=DEV)
    wide[:, 4] = ints([5, -1, 6])
    got = tm.paged_plan(ints([3, 3, 32]), ints([1, 1, 1]), wide[:, 4:8], ints([8, 9]), ints([2]), page_size=32, max_tokens=3)
    assert got.slots.tolist() == [5 * 32 + 3, -1, 9 * 32] and got.admitted.all()
    assert wide[2, 5] == 9 and (wide[:, 8:] == -7).all() and (wide[:, :4] == -7).all()


def test_plan_refusals():
    ok = dict(cached=ints([1]), new_tokens=ints([1]), block_table=ints([[1, 2]]), free_pages=ints([3]), free_count=ints([1]), page_size=32, max_tokens=1)
    for over, text in ((dict(cached=ints([1], torch.int64)), "dtype int32"), (dict(new_tokens=ints([1, 1])), "one entry for each request"),
                       (dict(block_table=ints([1, 2])), "2 dimensions"), (dict(free_count=ints([1, 2])), "one entry"), (dict(page_size=0), "positive"),
                       (dict(max_tokens=-1), "not be negative"), (dict(free_pages=torch.tensor([3], dtype=torch.int32)), "must be on"),
                       (dict(block_table=ints([[1, 2], [3, 4]]).t()[:1]), "contiguous rows")):
        with pytest.raises(RuntimeError, match=text):
            tm.paged_plan(**{**ok, **over})
    with pytest.raises(RuntimeError, match="at most 8192 requests"):
        tm.paged_plan(ints([0] * 8193), ints([0] * 8193), torch.zeros(8193, 1, dtype=torch.int32, device=DEV), ints([3]), ints([1]), page_size=32, max_tokens=1)


# ---- writes -----------------------------------------------------------------------------------------------------------
def _pool(P, page, H, D, block, form, seed, scale_power=-6):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(P, page, H, D, generator=g)
    x = (x * 100).clamp(-448, 448).to(F8) if form == F8 else (x * 40).round().clamp(-127, 127).to(I8)
    s = torch.exp2(torch.randint(scale_power - 2, scale_power + 3, (P, page // block, H), generator=g).float())
    return x, s if form == F8 else s * 0.7


def _check_write(key, value, slots, kp, vp, ks, vs, views=None):
    """Runs the call on device copies (or on the given views of them) and compares every byte of both pools and all scales."""
    dev = {n: t.to(DEV) for n, t in (("kp", kp), ("vp", vp), ("ks", ks), ("vs", vs))}
    dev.update(views or {})
    tm.paged_cache_write(key if key.is_cuda else key.to(DEV), value if value.is_cuda else value.to(DEV), dev["kp"], dev["vp"], dev["ks"], dev["vs"],
                         torch.as_tensor(slots, dtype=torch.int64, device=DEV))
    for x, p, s, gp, gs in ((key, kp, ks, dev["kp"], dev["ks"]), (value, vp, vs, dev["vp"], dev["vs"])):
        wp, ws = ref.write(x.double().cpu().numpy(), p.double().numpy(), s.numpy(), slots, p.dtype == I8)
        assert np.array_equal(gs.cpu().numpy(), ws)
        assert np.array_equal(gp.cpu().double().numpy(), wp, equal_nan=True)
    return dev


def _rows(T, H, D, dtype, seed, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, D, generator=g)
    if spread:
        x *= torch.exp2(torch.randint(-6, 7, (T, H, 1), generator=g).float())
    return x.to(dtype)


def _slots(starts, P, page, seed):
    """Slots of sequences that append n rows from position c on, each in pages of its own."""
    r = np.random.RandomState(seed)
    order, used, out = r.permutation(P), 0, []
    for c, n in starts:
        need = -(-(c + n) // page)
        pages = order[used:used + need]
        used += need
        assert used <= P
        out += [int(pages[p // page]) * page + p % page for p in range(c, c + n)]
    return out


@pytest.mark.parametrize("form", [F8, I8])
@pytest.mark.parametrize("dtype,D,H,page,block", [(BF, 128, 2, 64, 64), (HF, 64, 3, 128, 32), (BF, 96, 1, 32, 32), (HF, 256, 2, 96, 96), (BF, 16, 4, 256, 128),
                                                  (HF, 112, 5, 64, 32)])
@pytest.mark.parametrize("starts", [[(0, 1)], [(5, 1), (63, 1), (64, 1), (31, 1)], [(0, 64), (7, 90), (32, 33)], [(3, 300), (0, 1), (100, 150)]])
def test_write(form, dtype, D, H, page, block, starts):
    P = sum(-(-(c + n) // page) for c, n in starts) + 2
    slots = _slots(starts, P, page, D + page)
    T = len(slots)
    (kp, ks), (vp, vs) = _pool(P, page, H, D, block, form, 1), _pool(P, page, H, D, block, form, 2)
    _check_write(_rows(T, H, D, dtype, 3), _rows(T, H, D, dtype, 4), slots, kp, vp, ks, vs)


@pytest.mark.parametrize("form", [F8, I8])
def test_write_many_rows_with_padding_and_slots_outside_the_pool(form):
    """Long enough for the variant that looks for runs in chunks; padding in front, between and behind, and slots that the pool does
    not have, are left out."""
    page, block, H, D = 64, 32, 2, 128
    P = 30
    slots = _slots([(10, 500), (0, 257), (63, 1), (40, 600)], P, page, 5)
    slots = [-1] * 3 + slots[:182] + [-1] + slots[182:910] + [P * page, 2 ** 40, -2 ** 40, 2 ** 32 + 1] + slots[910:] + [-1] * 70  # cut between blocks
    T = len(slots)
    (kp, ks), (vp, vs) = _pool(P, page, H, D, block, form, 11), _pool(P, page, H, D, block, form, 12)
    _check_write(_rows(T, H, D, BF, 13), _rows(T, H, D, BF, 14), slots, kp, vp, ks, vs)
    # nothing but padding
    _check_write(_rows(9, H, D, BF, 13), _rows(9, H, D, BF, 14), [-1] * 9, kp, vp, ks, vs)


@pytest.mark.parametrize("form", [F8, I8])
@pytest.mark.parametrize("dtype,D,page,block", [(BF, 128, 128, 128), (HF, 256, 64, 64), (BF, 96, 256, 128), (HF, 64, 512, 256), (BF, 256, 512, 512), (HF, 16, 1024, 1024)])
def test_write_blocks_longer_than_a_wavefront_holds(form, dtype, D, page, block):
    """Whole blocks, parts of them at both ends, single rows and rows of many requests, in a call long enough for runs to be shared;
    infinities and NaN in some rows, blocks whose scale grows and blocks that keep theirs."""
    H, starts = 2, [(0, 700), (page - 3, 9), (5, 1), (block + 31, 300), (2 * page - 1, 1), (17, page)]
    P = sum(-(-(c + n) // page) for c, n in starts) + 2
    slots = _slots(starts, P, page, D + block)
    T = len(slots)
    slots = [-1] * 5 + slots + [-1] * 40
    (kp, ks), (vp, vs) = _pool(P, page, H, D, block, form, 15), _pool(P, page, H, D, block, form, 16)
    key, value = _rows(T + 45, H, D, dtype, 17), _rows(T + 45, H, D, dtype, 18)
    key[100, 0, 3], key[101, 1, 5], key[650, 0, 0], value[720, 1, D - 1] = math.inf, math.nan, -math.inf, math.nan
    value[800] = 0
    _check_write(key, value, slots, kp, vp, ks, vs)


@pytest.mark.parametrize("H,D,page,block", [(1, 16, 64, 32), (12, 16, 64, 64), (24, 16, 32, 32), (64, 16, 96, 96), (24, 64, 256, 256), (64, 64, 256, 256)])
def test_write_long_and_single_rows_among_one_another(H, D, page, block):
    """Runs that begin anywhere in the tokens that are looked through together, from one of them to 32, and end in others."""
    starts = [(9, 1), (0, 500)] + [(page * i + 7 * i, 1) for i in range(1, 40)] + [(1, 257), (block - 1, 2)] + [(5 * i, 3) for i in range(20)] + [(0, 513)]
    P = sum(-(-(c + n) // page) for c, n in starts) + 2
    slots = _slots(starts, P, page, H)
    slots = slots[:501] + [-1] * 33 + slots[501:]
    (kp, ks), (vp, vs) = _pool(P, page, H, D, block, F8, 33), _pool(P, page, H, D, block, F8, 34)
    _check_write(_rows(len(slots), H, D, BF, 35), _rows(len(slots), H, D, BF, 36), slots, kp, vp, ks, vs)


@pytest.mark.parametrize("form", [F8, I8])
def test_write_rows_of_a_block_in_any_order(form):
    page, block, H, D = 64, 64, 2, 64
    (kp, ks), (vp, vs) = _pool(4, page, H, D, block, form, 21), _pool(4, page, H, D, block, form, 22)
    slots = [130, 128 + 63, 128 + 5, 128 + 40] + [64 + 9, 64, 64 + 3]
    _check_write(_rows(7, H, D, HF, 23), _rows(7, H, D, HF, 24), slots, kp, vp, ks, vs)


@pytest.mark.parametrize("form", [F8, I8])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_write_of_special_values(form, dtype):
    """Zeros, infinities, NaN, the type's largest and smallest values, magnitudes on either side of a power of two's limit."""
    page = block = 32
    H, D = 2, 32
    big = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal
    T = 9
    x = torch.zeros(T, H, D, dtype=dtype)
    x[1, 0, 3], x[1, 1, 5] = math.inf, -math.inf     # nothing finite but zeros
    x[2, 0, :4] = torch.tensor([math.nan, 1.0, -math.inf, 448.0], dtype=dtype)
    x[3, 0], x[3, 1] = big, -big
    x[4, 0, 0], x[4, 1, 0] = tiny, tiny / 4
    x[5, 0, 0], x[5, 1, 0] = 448.0, 450.0            # 1.75 x 2^8 and the next bf16 (and fp16) values above it
    x[6, 0, :] = torch.linspace(-2, 2, D)
    x[7, 0, :8] = torch.tensor([448, 2 ** -6, 2 ** -9, 2 ** -10, 3 * 2 ** -10, 2 ** -11, 17, 19], dtype=dtype)  # ties and subnormals of e4m3
    x[8] = math.nan
    for first in (0, 4):  # the block's first row, and rows that join others
        slots = [i * page + first for i in range(T)]
        (kp, ks), (vp, vs) = _pool(T, page, H, D, block, form, 31), _pool(T, page, H, D, block, form, 32)
        _check_write(x, (x * 1).flip(2), slots, kp, vp, ks, vs)


@pytest.mark.parametrize("form", [F8, I8])
def test_write_starts_a_recycled_block_anew(form):
    """What a page held before, an enormous scale or NaN bytes, does not matter once its first slot is written."""
    page = block = 32
    H, D = 1, 32
    (kp, ks), (vp, vs) = _pool(3, page, H, D, block, form, 41), _pool(3, page, H, D, block, form, 42)
    ks[1], vs[1] = 1e30, math.inf
    kp.view(torch.uint8)[1] = 0x7f
    _check_write(_rows(5, H, D, BF, 43), _rows(5, H, D, BF, 44), [32, 33, 34, 35, 36], kp, vp, ks, vs)


def test_write_token_by_token_is_write_at_once_where_nothing_rounds_twice():
    """e4m3's scales are powers of two: rows appended one by one, scales growing on the way, come out as written at once as long as
    nothing becomes subnormal."""
    page = block = 64
    H, D, T = 2, 64, 64
    x = (torch.rand(T, H, D, generator=torch.Generator().manual_seed(1)) + 1).to(BF)
    x *= torch.exp2(torch.arange(T) // 10).to(BF)[:, None, None]
    x[:, :, ::2] *= -1
    def fresh():
        return [torch.zeros(2, page, H, D, dtype=torch.uint8, device=DEV).view(F8) for _ in range(2)] + [torch.zeros(2, 1, H, device=DEV) for _ in range(2)]
    a, b = fresh(), fresh()
    slots = torch.arange(64, 128, device=DEV)
    xd = x.to(DEV)
    tm.paged_cache_write(xd, -xd, *a, slots)
    for t in range(T):
        tm.paged_cache_write(xd[t:t + 1], -xd[t:t + 1], *b, slots[t:t + 1])
    for y, z in zip(a, b):
        assert torch.equal(y.view(torch.uint8), z.view(torch.uint8))


def test_write_strided_views():
    """Rows cut out of a fused projection, pools with padded rows and head-major pages, scales between other numbers."""
    page, block, H, D, T, P = 64, 32, 2, 64, 70, 5
    qkv = _rows(T, 8, D, BF, 51).to(DEV)
    key, value = qkv[:, 4:6], qkv[:, 6:8]
    (kp, ks), (vp, vs) = _pool(P, page, H, D, block, F8, 52), _pool(P, page, H, D, block, F8, 53)
    wide = torch.zeros(P, page, H, D + 16, dtype=torch.uint8, device=DEV).view(F8)
    wide.view(torch.uint8)[..., :D] = kp.view(torch.uint8).to(DEV)
    major = vp.to(DEV).view(torch.uint8).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3).view(F8)
    scales = torch.zeros(P, page // block, H, 3, device=DEV)
    scales[..., 1] = ks.to(DEV)
    slots = _slots([(10, 60), (0, 10)], P, page, 54)
    _check_write(key, value, slots, kp, vp, ks, vs, dict(kp=wide[..., :D], vp=major, ks=scales[..., 1]))
    assert not wide.view(torch.uint8)[..., D:].any() and not scales[..., 0].any() and not scales[..., 2].any()
    odd = torch.zeros(T, H, D + 1, dtype=BF, device=DEV)  # rows that 16-byte loads cannot take are copied
    odd[..., :D] = key
    _check_write(odd[..., :D], value, slots, kp, vp, ks, vs)


def test_write_refusals():
    f8 = torch.zeros(4, 64, 2, 64, dtype=torch.uint8, device=DEV).view(F8)
    sc = torch.zeros(4, 2, 2, device=DEV)
    x = torch.zeros(3, 2, 64, dtype=BF, device=DEV)
    s = ints([0, 1, 2], torch.int64)
    for args, text in (((x.float(), x.float(), f8, f8, sc, sc, s), "float16 or bfloat16"), ((x, x.half(), f8, f8, sc, sc, s), "same dtype"),
                       ((x, x, f8, f8, sc, sc, s.int()), "int64"), ((x, x, f8, f8, sc, sc, s[:2]), "int64"), ((x, x[:2], f8, f8, sc, sc, s), "tokens, heads"),
                       ((x, x, f8.view(I8), f8, sc, sc, s), "same dtype and shape"), ((x, x, f8.view(torch.uint8), f8, sc, sc, s), "float8_e4m3fn or int8"),
                       ((x, x, f8, f8, sc.half(), sc, s), "float32"), ((x, x, f8, f8, sc[:, :, :1], sc, s), "pages, blocks, heads"),
                       ((x, x, f8, f8, torch.zeros(4, 4, 2, device=DEV), torch.zeros(4, 4, 2, device=DEV), s), "multiple of 32 tokens"),
                       ((x[..., :40], x[..., :40], f8[..., :40], f8[..., :40], sc, sc, s), "multiple of 16"), ((x, x, f8[:0], f8[:0], sc[:0], sc[:0], s), "no pages"),
                       ((x, x, f8.cpu(), f8, sc, sc, s), "must be on"), ((x[:, :1], x[:, :1], f8, f8, sc, sc, s), "1 heads of 64"),
                       ((x.clone().requires_grad_(), x, f8, f8, sc, sc, s), "for inference")):
        with pytest.raises(RuntimeError, match=text):
            tm.paged_cache_write(*args)
    tm.paged_cache_write(x[:0], x[:0], f8, f8, sc, sc, s[:0])  # no rows: nothing happens


# ---- attention --------------------------------------------------------------------------------------------------------
def _cache_for(lens, page, H, D, block, form, seed, extra=2):
    """A pool with finite values everywhere a sequence reaches and NaN (e4m3) or 127 elsewhere, its scales, and the table."""
    width = max(1, -(-max(lens) // page))
    P = len(lens) * width + extra
    (kp, ks), (vp, vs) = _pool(P, page, H, D, block, form, seed, -8), _pool(P, page, H, D, block, form, seed + 1, -8)
    table = torch.randperm(P, generator=torch.Generator().manual_seed(seed))[:len(lens) * width].reshape(len(lens), width).to(torch.int32)
    live = torch.zeros(P * page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for r in range(n):
            live[int(table[b, r // page]) * page + r % page] = True
    for p in (kp, vp):
        p.view(torch.uint8).view(P * page, H, D)[~live] = 0x7f
    return kp, vp, ks, vs, table


def _check_attention(q, kp, vp, ks, vs, table, lens, causal, scale=None, cu=None, max_q=None, views=None, **more):
    """q [B, Hq, Sq, D], or packed [T, Hq, D] with cu; all on the CPU."""
    v = views or {}
    args = [v.get("q", q.to(DEV)), v.get("kp", kp.to(DEV)), v.get("vp", vp.to(DEV)), v.get("table", table.to(DEV)), ints(lens)]
    if cu is not None:
        more = dict(more, cu_seqlens_q=ints(cu), max_seqlen_q=max_q)
    out, lse = tm.paged_attention(*args, is_causal=causal, scale=scale, key_scales=v.get("ks", ks.to(DEV)), value_scales=v.get("vs", vs.to(DEV)), **more)
    D = q.shape[-1]
    assert out.shape == q.shape and out.dtype == q.dtype
    assert lse.shape == ((q.shape[1], q.shape[0]) if cu is not None else q.shape[:3]) and lse.dtype == torch.float32
    got, gl = out.double().cpu(), lse.double().cpu()
    for b, n in enumerate(lens):
        n = min(max(n, 0), table.shape[1] * kp.shape[1])
        rows = q[cu[b]:cu[b + 1]] if cu is not None else q[b].transpose(0, 1)
        o, z, tol, ltol = ref.attention(rows.double(), (kp, vp), (ks, vs), table[b], n, causal, scale if scale is not None else 1 / math.sqrt(D),
                                        torch.finfo(q.dtype).eps)
        g = got[cu[b]:cu[b + 1]] if cu is not None else got[b].transpose(0, 1)
        l = gl[:, cu[b]:cu[b + 1]].T if cu is not None else gl[b].T
        bad = ~((g - o).abs() <= tol)
        assert not bad.any(), (b, float((g - o).abs().max()), float(tol.max()), bad.nonzero()[:3].tolist())
        dead = torch.isinf(z)
        assert torch.equal(torch.isinf(l), dead) and (l[dead] > 0).all()
        assert ((l - z).abs()[~dead] <= ltol[~dead]).all(), float((l - z).abs()[~dead].max())
    return out, lse


def _q(shape, dtype, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype,form", [(BF, F8), (HF, I8), (HF, F8), (BF, I8)])
@pytest.mark.parametrize("D,page,block", [(128, 64, 64), (64, 128, 32), (256, 32, 32), (96, 96, 32), (16, 64, 64), (208, 256, 128)])
@pytest.mark.parametrize("Sq,group", [(1, 1), (1, 4), (3, 7), (2, 16), (5, 1), (40, 3)])
def test_attention_shapes(dtype, form, D, page, block, Sq, group):
    lens = [1 + Sq, 5 * page + 17, page, 0, 2 * page + 1, Sq]
    kp, vp, ks, vs, table = _cache_for(lens, page, 2, D, block, form, D + page + Sq)
    _check_attention(_q((6, 2 * group, Sq, D), dtype, 7), kp, vp, ks, vs, table, lens, True)


@pytest.mark.parametrize("form", [F8, I8])
@pytest.mark.parametrize("lens", [[1], [31, 32, 33], [64, 65, 0], [2000, 1, 777]])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_lengths(form, lens, causal):
    kp, vp, ks, vs, table = _cache_for(lens, 64, 1, 64, 32, form, 61)
    _check_attention(_q((len(lens), 8, 1, 64), BF, 8), kp, vp, ks, vs, table, lens, causal)
    _check_attention(_q((len(lens), 2, 9, 64), HF, 9), kp, vp, ks, vs, table, lens, causal)  # rows that see no key among them


@pytest.mark.parametrize("dtype,form", [(BF, F8), (HF, I8)])
@pytest.mark.parametrize("D,heads,kv_heads", [(128, 8, 2), (64, 6, 1), (256, 4, 2)])
def test_attention_packed(dtype, form, D, heads, kv_heads):
    """Prompts, chunks deep in a cache, decodes and idle sequences in one call; rows behind the last sequence stay out of it."""
    rows, lens = [70, 1, 0, 130, 1, 5], [70, 900, 50, 500, 1, 4]   # the last has fewer keys than rows
    cu = [0]
    for n in rows:
        cu.append(cu[-1] + n)
    kp, vp, ks, vs, table = _cache_for(lens, 64, kv_heads, D, 32, form, 71)
    q = _q((cu[-1], heads, D), dtype, 10)
    for max_q in (130, 400):
        _check_attention(q, kp, vp, ks, vs, table, lens, True, cu=cu, max_q=max_q)
    _check_attention(q, kp, vp, ks, vs, table, lens, False, cu=cu, max_q=130)


@pytest.mark.parametrize("B", [1, 64, 65, 130])
def test_attention_packed_batches_of_every_kind(B):
    """No rows, one, as many as a wavefront of the tile kernel holds, one more, a block and its neighbours; both ways to find a
    sequence, in one slice and in several (few heads and long tables)."""
    g = np.random.RandomState(B)
    new = [int(x) for x in g.choice((0, 1, 1, 1, 8, 9, 31, 32, 33, 64, 130), B)]
    new[-1] = 150
    for keys, heads, kv_heads in ((200, 8, 2), (3000 if B > 1 else 9000, 4, 1)):
        lens = [max(n, int(g.randint(1, keys))) for n in new]
        cu = [0] + [int(x) for x in np.cumsum(new)]
        kp, vp, ks, vs, table = _cache_for(lens, 64, kv_heads, 64, 64, F8, 75)
        _check_attention(_q((cu[-1], heads, 64), BF, 16), kp, vp, ks, vs, table, lens, True, cu=cu, max_q=150)


def test_attention_packed_leaves_other_rows_alone():
    """C ABI: rows behind the last sequence, and rows beyond seqlen_q, keep what they hold; cu_seqlens beyond the rows are clipped."""
    import ctypes

    from torch_mlu_amd import capi_kv

    lens, cu, D, H = [100, 40], [0, 20, 23], 64, 2
    kp, vp, ks, vs, table = (t.to(DEV) for t in _cache_for(lens, 32, 1, D, 32, F8, 81))
    q = _q((30, H, D), BF, 11).to(DEV)
    full, flse = tm.paged_attention(q, kp, vp, table, ints(lens), is_causal=True, key_scales=ks, value_scales=vs, cu_seqlens_q=ints(cu), max_seqlen_q=20)
    for seqlen, cut, splits in ((20, cu, 1), (20, cu, 3), (12, cu, 1), (12, cu, 3), (20, [0, 20, 2 ** 30], 1), (20, [-5, 20, 23], 2)):
        out, lse = torch.full_like(q, 7.0), torch.full((H, 30), 7.0, device=DEV)
        p = capi_kv.FaKvAttnParams()
        cud, used = ints(cut), ints(lens)
        for n, t in (("q", q), ("key_pages", kp), ("value_pages", vp), ("key_scales", ks), ("value_scales", vs), ("out", out), ("lse", lse),
                     ("block_table", table), ("seqused_k", used), ("cu_seqlens_q", cud)):
            setattr(p, n, t.data_ptr())
        p.q_stride_s = p.o_stride_s = H * D
        p.q_stride_h = p.o_stride_h = D
        for n, t in (("kp", kp), ("vp", vp)):
            for d, i in zip("psh", range(3)):
                setattr(p, f"{n}_stride_{d}", t.stride(i))
        for n, t in (("ks", ks), ("vs", vs)):
            for d, i in zip("pbh", range(3)):
                setattr(p, f"{n}_stride_{d}", t.stride(i))
        p.lse_stride_h, p.lse_stride_s, p.block_table_stride = 30, 1, table.shape[1]
        p.batch, p.heads_q, p.heads_k, p.seqlen_q, p.total_q, p.head_dim = 2, H, 1, seqlen, 30, D
        p.num_pages, p.table_pages, p.page_size, p.scale_block = kp.shape[0], table.shape[1], 32, 32
        p.scale, p.dtype, p.format, p.is_causal, p.num_splits = D ** -0.5, 1, 0, 1, splits
        need = capi_kv.lib().fa_kv_attn_workspace_bytes(ctypes.byref(p))
        ws = torch.full((need // 4 + 4,), float("nan"), device=DEV)  # a slot read before it is written would show
        assert capi_kv.lib().fa_kv_attn_launch(ctypes.byref(p), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        first = min(20, seqlen)
        assert (out[first:20] == 7).all() and (lse[:, first:20] == 7).all()
        if cut == cu:
            assert (out[23:] == 7).all() and (lse[:, 23:] == 7).all()
            assert torch.allclose(out[:first].float(), full[:first].float(), atol=2e-2) and torch.allclose(lse[:, :first], flse[:, :first], atol=1e-4)
        assert torch.isfinite(out).all()


def test_attention_of_long_caches_in_slices():
    """Splits of the key range, among them slices that one sequence has and another has not, against the definition."""
    lens = [9000, 300, 0, 4097]
    for dtype, form, Sq, heads in ((BF, F8, 1, 8), (HF, I8, 3, 4), (BF, F8, 33, 2)):
        kp, vp, ks, vs, table = _cache_for(lens, 128, 2, 128, 64, form, 91)
        _check_attention(_q((4, heads, Sq, 128), dtype, 12), kp, vp, ks, vs, table, lens, True)


def test_attention_entries_outside_the_pool_hide_their_keys():
    lens = [300, 200, 64]
    kp, vp, ks, vs, table = _cache_for(lens, 64, 2, 64, 32, F8, 101)
    table[0, 1], table[0, 3], table[1, 0], table[2, 0] = -1, kp.shape[0], 2 ** 31 - 1, -2 ** 31
    for Sq in (1, 20):
        _check_attention(_q((3, 4, Sq, 64), BF, 13), kp, vp, ks, vs, table, lens, True)


def test_attention_lengths_beyond_the_table_and_below_zero():
    lens = [128, 64]
    kp, vp, ks, vs, table = _cache_for(lens, 64, 1, 64, 64, I8, 111)
    kp.fill_(3), vp.fill_(5)
    _check_attention(_q((2, 4, 2, 64), HF, 14), kp, vp, ks, vs, table, [2 ** 31 - 1, -3], False)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_attention_scales(scale):
    """Softmax scales of either sign and 0, blocks whose scales differ by 2^40 and blocks with scale 0, either type."""
    lens = [500, 33]
    for dtype, form in ((BF, F8), (HF, I8), (HF, F8)):
        kp, vp, ks, vs, table = _cache_for(lens, 64, 2, 64, 32, form, 121)
        vs *= torch.exp2(torch.randint(-20, 3, vs.shape, generator=torch.Generator().manual_seed(3)).float())
        ks[::3] = 0.0
        vs[1::3] = 0.0
        for Sq in (1, 12):
            _check_attention(_q((2, 4, Sq, 64), dtype, 15) * 0.25, kp, vp, ks, vs, table, lens, True, scale=scale)


def test_attention_large_scores():
    """Scores in the thousands: one key has it all; a later block's score moves the maximum far."""
    lens = [700]
    kp, vp, ks, vs, table = _cache_for(lens, 64, 1, 64, 32, F8, 131)
    q = _q((1, 4, 2, 64), BF, 16) * 30
    _check_attention(q, kp, vp, ks * 64, vs, table, lens, True)


@pytest.mark.parametrize("Sq,heads,D", [(4, 4, 64), (4, 8, 128), (6, 16, 128), (3, 4, 256), (70, 4, 64), (200, 2, 128), (150, 2, 256)])
@pytest.mark.parametrize("splits_keys", [300, 5000])
def test_attention_nan_in_keys_that_some_rows_do_not_see(Sq, heads, D, splits_keys):
    """NaN rows of K and V at some of the call's own tokens: the rows before them do not know, the rows from them on are NaN, and lse
    of a NaN in V alone is what it is."""
    n = splits_keys + Sq
    kp, vp, ks, vs, table = _cache_for([n, 40 + Sq], 64, 2, D, 32, F8, 135)
    q = _q((2, heads, Sq, D), BF, 20)
    good, gl = tm.paged_attention(q.to(DEV), kp.to(DEV), vp.to(DEV), table.to(DEV), ints([n, 40 + Sq]), is_causal=True, key_scales=ks.to(DEV), value_scales=vs.to(DEV))
    first = Sq - Sq // 3 - 1  # the token, in the call, whose row is NaN
    for which in (kp, vp):
        bad = [t.clone() for t in (kp, vp)]
        target = bad[0] if which is kp else bad[1]
        pos = n - Sq + first
        target.view(torch.uint8)[int(table[0, pos // 64]), pos % 64] = 0xff
        out, lse = tm.paged_attention(q.to(DEV), bad[0].to(DEV), bad[1].to(DEV), table.to(DEV), ints([n, 40 + Sq]), is_causal=True, key_scales=ks.to(DEV),
                                      value_scales=vs.to(DEV))
        assert torch.equal(out[1], good[1]) and torch.equal(lse[1], gl[1])
        assert torch.equal(out[0, :, :first], good[0, :, :first]) and torch.equal(lse[0, :, :first], gl[0, :, :first])
        assert torch.isnan(out[0, :, first:]).all()
        assert torch.isnan(lse[0, :, first:]).all() if which is kp else torch.equal(lse[0, :, first:], gl[0, :, first:])


def test_attention_nan_in_a_query_row():
    lens = [500, 90]
    kp, vp, ks, vs, table = (t.to(DEV) for t in _cache_for(lens, 64, 2, 64, 32, F8, 136))
    for Sq in (3, 40):
        q = _q((2, 4, Sq, 64), BF, 21).to(DEV)
        kw = dict(is_causal=True, key_scales=ks, value_scales=vs)
        good, gl = tm.paged_attention(q, kp, vp, table, ints(lens), **kw)
        q[0, 1, 2, 5] = math.nan
        out, lse = tm.paged_attention(q, kp, vp, table, ints(lens), **kw)
        assert torch.isnan(out[0, 1, 2]).all() and torch.isnan(lse[0, 1, 2])
        out[0, 1, 2], lse[0, 1, 2] = good[0, 1, 2], gl[0, 1, 2]
        assert torch.equal(out, good) and torch.equal(lse, gl)


def test_attention_strided_views():
    lens, page, H, D = [200, 90], 64, 2, 64
    kp, vp, ks, vs, table = _cache_for(lens, page, H, D, 32, F8, 141)
    P = kp.shape[0]
    wide = torch.zeros(P, page, H, D + 16, dtype=torch.uint8, device=DEV).view(F8)
    wide.view(torch.uint8)[..., :D] = kp.view(torch.uint8).to(DEV)
    major = vp.to(DEV).view(torch.uint8).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3).view(F8)
    scales = torch.zeros(P, 2, H, 2, device=DEV)
    scales[..., 1] = ks.to(DEV)
    tbl = torch.full((2, 9), -1, dtype=torch.int32, device=DEV)
    tbl[:, 3:3 + table.shape[1]] = table.to(DEV)
    q = _q((2, 8, 3, D), BF, 17)
    fused = torch.zeros(2, 3, 12, D, dtype=BF, device=DEV)
    fused[:, :, 2:10] = q.transpose(1, 2).to(DEV)
    odd = torch.zeros(2, 8, 3, D + 1, dtype=BF, device=DEV)
    odd[..., :D] = q.to(DEV)
    views = dict(kp=wide[..., :D], vp=major, ks=scales[..., 1], table=tbl[:, 3:3 + table.shape[1]])
    for qv in (fused[:, :, 2:10].transpose(1, 2), odd[..., :D]):
        _check_attention(q, kp, vp, ks, vs, table, lens, True, views=dict(views, q=qv))


def test_attention_pool_beyond_32_bit_offsets():
    """Pages whose bytes lie past 2^32 from the pool's start."""
    page, H, D = 64, 8, 128
    P = (5 << 30) // (page * H * D)
    pool = torch.zeros(P, page, H, D, dtype=torch.uint8, device=DEV)
    scales = torch.full((P, 1, H), 2.0 ** -7, device=DEV)
    lens = [300, 100]
    kp, vp, ks, vs, table = _cache_for(lens, page, H, D, 64, F8, 151)
    n = kp.shape[0]
    for shift in (P - n, P // 2):
        far = table + shift
        k, v = pool.clone() if shift == P // 2 else pool, pool
        k[shift:shift + n] = kp.view(torch.uint8).to(DEV)
        scales[shift:shift + n] = ks.to(DEV)
        q = _q((2, 16, 1, D), BF, 18)
        out, lse = tm.paged_attention(q.to(DEV), k.view(F8), k.view(F8), far.to(DEV), ints(lens), key_scales=scales, value_scales=scales)
        near = tm.paged_attention(q.to(DEV), kp.to(DEV), kp.to(DEV), table.to(DEV), ints(lens), key_scales=ks.to(DEV), value_scales=ks.to(DEV))
        assert torch.equal(out, near[0]) and torch.equal(lse, near[1])
        # and a row written there
        x = _q((1, H, D), BF, 19).to(DEV)
        slot = torch.tensor([(shift + n - 1) * page], device=DEV)
        tm.paged_cache_write(x, x, k.view(F8), k.view(F8), scales, scales, slot)
        s = scales[shift + n - 1, 0].cpu().numpy()
        want = ref.e4m3(x[0].double().cpu().numpy() / s[:, None])
        assert np.array_equal(k[shift + n - 1, 0].view(F8).double().cpu().numpy(), want)
        if shift == P - n:
            pool.zero_()


def test_attention_without_rows_keys_or_sequences():
    kp, vp, ks, vs, table = (t.to(DEV) for t in _cache_for([64], 64, 2, 64, 64, F8, 161))
    kw = dict(key_scales=ks, value_scales=vs)
    z = lambda *s: torch.zeros(*s, dtype=BF, device=DEV)  # noqa: E731
    out, lse = tm.paged_attention(z(0, 4, 1, 64), kp, vp, table[:0], ints([]), **kw)
    assert out.shape == (0, 4, 1, 64) and lse.shape == (0, 4, 1)
    out, lse = tm.paged_attention(z(1, 4, 0, 64), kp, vp, table, ints([64]), **kw)
    assert out.shape == (1, 4, 0, 64)
    out, lse = tm.paged_attention(z(1, 4, 2, 64) + 1, kp, vp, table[:, :0], ints([64]), **kw)
    assert not out.any() and (lse == math.inf).all()
    out, lse = tm.paged_attention(z(0, 4, 64), kp, vp, table, ints([64]), cu_seqlens_q=ints([0, 0]), max_seqlen_q=0, **kw)
    assert out.shape == (0, 4, 64) and lse.shape == (4, 0)


def test_attention_refusals():
    kp, vp, ks, vs, table = (t.to(DEV) for t in _cache_for([64], 64, 2, 64, 64, F8, 171))
    q = torch.zeros(1, 4, 1, 64, dtype=BF, device=DEV)
    ok = dict(query=q, key_pages=kp, value_pages=vp, block_table=table, seqused_k=ints([64]), key_scales=ks, value_scales=vs)
    for over, text in ((dict(query=q.float()), "float16 or bfloat16"), (dict(query=q[0]), "query must be"), (dict(query=q[:, :3]), "must divide"),
                       (dict(seqused_k=ints([64, 1])), "one entry for each"), (dict(seqused_k=ints([64], torch.int64)), "int32"),
                       (dict(block_table=table.long()), "int32"), (dict(max_seqlen_q=3), "goes with"), (dict(cu_seqlens_q=ints([0, 1])), "packed|tokens, heads"),
                       (dict(query=q[:, :, 0], cu_seqlens_q=ints([0, 1])), "max_seqlen_q"), (dict(value_scales=vs[:1]), "pages, blocks, heads"),
                       (dict(query=q.clone().requires_grad_()), "for inference"), (dict(query=torch.zeros(1, 4, 1, 32, dtype=BF, device=DEV)), "heads of 32"),
                       (dict(key_pages=kp.cpu()), "must be on")):
        with pytest.raises(RuntimeError, match=text):
            tm.paged_attention(**{**ok, **over})


def test_cache_tensors_that_want_gradients_are_refused():
    """Neither operator has a gradient, so a scale that requires one would get none without a word."""
    kp, vp, ks, vs, table = (t.to(DEV) for t in _cache_for([64], 64, 2, 64, 64, F8, 172))
    q, x, slot = torch.zeros(1, 4, 1, 64, dtype=BF, device=DEV), torch.zeros(1, 2, 64, dtype=BF, device=DEV), ints([0], torch.int64)
    for i in range(2):
        scales = [ks, vs]
        scales[i] = scales[i].clone().requires_grad_()
        with pytest.raises(RuntimeError, match="for inference"):
            tm.paged_attention(q, kp, vp, table, ints([64]), key_scales=scales[0], value_scales=scales[1])
        with pytest.raises(RuntimeError, match="for inference"):
            tm.paged_cache_write(x, x, kp, vp, *scales, slot)
        with torch.no_grad():
            tm.paged_attention(q, kp, vp, table, ints([64]), key_scales=scales[0], value_scales=scales[1])


# ---- together -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("form,dtype", [(F8, BF), (I8, HF)])
def test_serving_loop(form, dtype):
    """Prompts, then decode steps, of requests that come and go: positions turned, rows written, attention read, step after step;
    each stage against its definition on the stage before it, and the cache against what went into it."""
    page, block, Hq, Hk, D, width, P = 64, 32, 8, 2, 64, 8, 40
    g = torch.Generator().manual_seed(5)
    kp, vp = (torch.full((P, page, Hk, D), 0x7f, dtype=torch.uint8, device=DEV).view(form) for _ in range(2))
    ks, vs = (torch.full((P, page // block, Hk), 1e30, device=DEV) for _ in range(2))
    table = torch.full((4, width), -1, dtype=torch.int32, device=DEV)
    free, count, cached = torch.randperm(P, generator=g).to(torch.int32).to(DEV), ints([P]), ints([0] * 4)
    freq, axes = tm.rotary_frequencies((16, 8, 8), device=DEV)
    held = [[torch.zeros(0, Hk, D) for _ in range(4)] for _ in range(2)]
    for step, new in enumerate([[70, 0, 33, 1], [1, 128, 1, 0], [1, 1, 1, 1], [1, 1, 64, 1], [2, 3, 1, 4]]):
        T = sum(new) + 3
        p = tm.paged_plan(cached, ints(new), table, free, count, page_size=page, max_tokens=T)
        assert p.admitted.all()
        q, k, v = (torch.randn(T, h, D, generator=g).to(dtype).to(DEV) for h in (Hq, Hk, Hk))
        pos = torch.stack([p.positions, p.positions // 8, p.positions % 8])
        qr, kr = tm.rotary(q, k, pos, freq, axes)
        want, tol = ref.rotary(k.double().cpu(), pos.cpu(), freq.cpu(), axes.cpu(), False)
        assert ((kr.double().cpu() - want).abs() <= tol + want.abs() * torch.finfo(dtype).eps / 2).all()
        tm.paged_cache_write(kr, v, kp, vp, ks, vs, p.slots)
        out, lse = tm.paged_attention(qr, kp, vp, table, p.seqused_k, is_causal=True, key_scales=ks, value_scales=vs, cu_seqlens_q=p.cu_seqlens,
                                      max_seqlen_q=max(new))
        cu = p.cu_seqlens.tolist()
        for b in range(4):
            n = int(p.seqused_k[b])
            for i, (x, pages, sc) in enumerate(((kr, kp, ks), (v, vp, vs))):
                held[i][b] = torch.cat([held[i][b], x[cu[b]:cu[b + 1]].float().cpu()])
                assert len(held[i][b]) == n
                if n:
                    back, _ = ref.gathered(pages.cpu(), sc.cpu(), table[b].cpu(), n)
                    # a row is rounded once to half a step and at most once more each time its block's scale grows, a block's scale
                    # at most doubling what the largest row needs: e4m3 2^-4 relative and half a subnormal step, int8 half a step
                    top = torch.stack([held[i][b][j // block * block:j // block * block + block].abs().amax((0, 2)) for j in range(n)])
                    rounds = 4
                    near = held[i][b].abs() * 2.0 ** -4 + top[:, :, None] * (2.0 ** -17 * rounds if form == F8 else 1.001 / 254 * rounds)
                    if form == I8:
                        near = top[:, :, None] * (1.001 / 254 * rounds)
                    assert ((back - held[i][b].double()).abs() <= near).all()
            o, z, tol, ltol = ref.attention(qr[cu[b]:cu[b + 1]].double().cpu(), (kp.cpu(), vp.cpu()), (ks.cpu(), vs.cpu()), table[b].cpu(), n, True, D ** -0.5,
                                            torch.finfo(dtype).eps)
            assert ((out[cu[b]:cu[b + 1]].double().cpu() - o).abs() <= tol).all()
            assert ((lse[:, cu[b]:cu[b + 1]].T.double().cpu() - z).abs() <= ltol).all()
        cached, count = p.seqused_k, p.free_count
        if step == 2:  # request 1 ends, its pages go back, another takes its place
            pages = -(-int(cached[1]) // page)
            c = int(count)
            free[c:c + pages] = table[1, :pages]
            count = count + pages
            cached = cached.clone()
            cached[1] = 0
            table[1] = -1
            held[0][1] = held[1][1] = torch.zeros(0, Hk, D)
    assert int(count) == P - sum(-(-int(n) // page) for n in cached)


def _step(s):
    p = tm.paged_plan(s["cached"], s["new"], s["table"], s["free"], s["count"], page_size=64, max_tokens=s["q"].shape[0])
    q, k = tm.rotary(s["q"], s["k"], p.positions[None], s["freq"], s["axes"])
    tm.paged_cache_write(k, s["v"], s["kp"], s["vp"], s["ks"], s["vs"], p.slots)
    out, lse = tm.paged_attention(q, s["kp"], s["vp"], s["table"], p.seqused_k, is_causal=True, key_scales=s["ks"], value_scales=s["vs"],
                                  cu_seqlens_q=p.cu_seqlens, max_seqlen_q=4)
    return list(p) + [q, k, out, lse]


def _state(seed, B=6):
    g = torch.Generator().manual_seed(seed)
    lens = [1000, 64, 130, 5, 700, 63][:B]
    kp, vp, ks, vs, table = (t.to(DEV) for t in _cache_for([n + 200 for n in lens], 64, 2, 64, 32, F8, seed))
    table = torch.cat([table, torch.full((B, 2), -1, dtype=torch.int32, device=DEV)], 1)
    freq, axes = tm.rotary_frequencies((32,), device=DEV)
    rnd = lambda h: torch.randn(20, h, 64, generator=g).to(BF).to(DEV)  # noqa: E731
    return dict(kp=kp, vp=vp, ks=ks, vs=vs, table=table, cached=ints(lens), new=ints([1, 2, 1, 4, 1, 3][:B]), free=ints(list(range(8))), count=ints([8]), q=rnd(8),
                k=rnd(2), v=rnd(2), freq=freq, axes=axes)


def test_step_in_a_graph():
    """A step captured once and replayed on other requests' data, eager work between the replays; every replay has the eager bits,
    also where two graphs take turns."""
    def clone(s):
        return {n: t.clone() for n, t in s.items()}

    def load(static, s):
        for n in static:
            static[n].copy_(s[n])

    statics = [clone(_state(1)), clone(_state(1))]
    graphs, outs = [], []
    for st in statics:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(st)
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(_step(st))
        graphs.append(gr)
    for i, seed in enumerate((2, 3, 4, 5, 6)):
        s = _state(seed)
        want_state = clone(s)
        want = _step(want_state)
        torch.cuda.synchronize()
        load(statics[i % 2], s)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        n = int(want[0][-1])
        for a, b in zip(outs[i % 2], want):
            if a.dim() == 3 and a.dtype == BF and a.shape[1] == 8:
                a, b = a[:n], b[:n]   # rows behind the last sequence are not written
            if a.dtype == torch.float32:
                a, b = a[:, :n], b[:, :n]
            assert torch.equal(a, b)
        for m in ("kp", "vp", "ks", "vs", "table"):
            assert torch.equal(statics[i % 2][m].view(torch.uint8), want_state[m].view(torch.uint8)), m


def test_step_on_another_stream_and_twice_at_once():
    a, b = _state(11), _state(12)
    wa, wb = _state(11), _state(12)
    ra, rb = _step(wa), _step(wb)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s1):
        ga = _step(a)
    with torch.cuda.stream(s2):
        gb = _step(b)
    torch.cuda.synchronize()
    for got, want in ((ga, ra), (gb, rb)):
        n = int(want[0][-1])
        assert torch.equal(got[-2][:n], want[-2][:n]) and torch.equal(got[-1][:, :n], want[-1][:, :n]) and torch.equal(got[3], want[3])
