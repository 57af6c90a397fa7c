"""The decode operators on the GPU against plain torch in 64 bits
(oracle/decode_ref.py): rotary positions, the page pool, attention over it, and a
decode loop of them together.

Tolerances. u = 2^-24 is fp32's half step. A rotated value has its cosine and sine
rounded once (u each), one product and one fused sum (u each) of |x_a| + |x_b|
times the gain: 4 u of that at most; a 16-bit result adds its own half step.
Pool rows are bit-exact. Attention: a score is a chain of at most D sums (D u of
sum |q k| scale, "reach"), a few roundings of the score itself and the
exponential; every weight is off by that, twice (numerator and sum); sums run over
chains of n positions; weights may be carried as two 16-bit parts where the queries
have 16 bits (2^-16). The bound is that factor times sum p |v|, plus the result's half step.
"""

import copy
import math
import pickle

import numpy as np
import pytest
import torch

from helpers import bits
from oracle import decode_ref as R
from shadowinfer_amd import KVPagePool, RotaryEmbedding, RotaryScaling, paged_attention
from shadowinfer_amd.shadowkv import PagedKVStore

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF_STEP = {F32: U, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}  # steps near zero


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


# ------------------------------------------------------------------- rotary
def check_rotated(got, x, positions, rope, transpose=False):
    n = rope.rotary_dim // 2
    inter = rope.layout == "interleaved"
    angles = torch.tensor(rope.angles, dtype=torch.float64)
    want = R.rotate(x, positions, angles, rope.value_factor, inter, transpose)
    size = R.rotate_magnitude(x, n, rope.value_factor, inter)
    # angles of far positions: p * f carries fp64's rounding, twice
    far = positions.double().abs().max() * max(rope.angles) * 2.0 ** -52 if positions.numel() else 0.0
    tol = size * (4 * U + far)
    tol = tol + HALF_STEP[x.dtype] * (want.abs() + tol) + TINY[x.dtype]
    tol[..., 2 * n:] = 0  # the rest is copied
    assert got.dtype == x.dtype and got.shape == x.shape
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D,rot", [(128, 128), (64, 32), (80, 32), (80, 80), (10, 6), (45, 44), (256, 64),
                                   (4, 2), (1024, 1024)])
@pytest.mark.parametrize("T", [1, 37])
def test_rotary_rows(dtype, layout, D, rot, T):
    g = gen(D * 7 + rot + T)
    rope = RotaryEmbedding(D, rotary_dim=rot, layout=layout)
    q, k = randn(g, T, 5, D, dtype=dtype), randn(g, T, 2, D, dtype=dtype)
    pos = torch.randint(0, 5000, (T,), generator=g, device="cuda")
    gq, gk = rope(pos, q, k)
    check_rotated(gq, q, pos, rope)
    check_rotated(gk, k, pos, rope)
    # q alone, other position type, in place: the same bits
    assert torch.equal(rope(pos.int(), q), gq)
    q2, k2 = q.clone(), k.clone()
    r = rope(pos, q2, k2, inplace=True)
    assert r[0] is q2 and r[1] is k2 and torch.equal(q2, gq) and torch.equal(k2, gk)


@pytest.mark.parametrize("tokens", [511, 2049, 5000])
def test_rotary_many_tokens(tokens):
    """Blocks of several tokens, the last one partly filled."""
    g = gen(tokens)
    rope = RotaryEmbedding(64, layout="half")
    q, k = randn(g, tokens, 3, 64, dtype=BF16), randn(g, tokens, 1, 64, dtype=BF16)
    pos = torch.randperm(tokens, generator=g, device="cuda")
    gq, gk = rope(pos, q, k)
    check_rotated(gq, q, pos, rope)
    check_rotated(gk, k, pos, rope)


def test_rotary_strides_batches_and_alignment():
    g = gen(1)
    B, S, Hq, Hk, D = 3, 17, 6, 2, 64
    rope = RotaryEmbedding(D)
    # columns of one projection
    x = randn(g, B, S, (Hq + 2 * Hk) * D, dtype=BF16)
    q = x[..., :Hq * D].unflatten(-1, (Hq, D))
    k = x[..., Hq * D:(Hq + Hk) * D].unflatten(-1, (Hk, D))
    pos = torch.randint(-50, 5000, (B, S), generator=g, device="cuda")
    gq, gk = rope(pos, q, k)
    check_rotated(gq, q, pos, rope)
    check_rotated(gk, k, pos, rope)
    # positions of one row for every batch row, and a strided position tensor
    row = torch.arange(2 * S, device="cuda")[::2]
    assert torch.equal(rope(row, q), rope(row.expand(B, S).contiguous(), q))
    # heads before tokens
    h = randn(g, B, Hq, S, D, dtype=F16)
    out = rope(pos, h.transpose(1, 2))
    check_rotated(out, h.transpose(1, 2), pos, rope)
    # in place on a projection's columns: the other columns stay
    y = x.clone()
    rope(pos, y[..., :Hq * D].unflatten(-1, (Hq, D)), y[..., Hq * D:(Hq + Hk) * D].unflatten(-1, (Hk, D)),
         inplace=True)
    assert torch.equal(y[..., :Hq * D].unflatten(-1, (Hq, D)), gq)
    assert torch.equal(y[..., (Hq + Hk) * D:], x[..., (Hq + Hk) * D:])
    # rows that no 16-byte load may touch, and a last dimension that is not contiguous
    flat = randn(g, S * Hq * D + 1, dtype=BF16)
    odd = flat[1:].view(S, Hq, D)
    assert torch.equal(rope(row, odd), rope(row, odd.clone()))
    turned = randn(g, S, D, Hq, dtype=BF16).transpose(1, 2)
    assert torch.equal(rope(row, turned), rope(row, turned.contiguous()))
    # one token for every head and batch row (stride 0)
    one = randn(g, 1, 1, D).expand(S, Hq, D)
    check_rotated(rope(row, one), one, row, rope)


@pytest.mark.parametrize("kind", ["linear", "ntk", "yarn", "bands"])
def test_rotary_scalings_and_transpose(kind):
    g = gen(5)
    rope = RotaryEmbedding(128, rotary_dim=64, base=500000.0, layout="interleaved",
                           scaling=RotaryScaling(kind, 16.0, original_positions=8192))
    x = randn(g, 50, 4, 128)
    pos = torch.randint(0, 131072, (50,), generator=g, device="cuda")
    check_rotated(rope(pos, x), x, pos, rope)
    check_rotated(rope(pos, x, transpose=True), x, pos, rope, transpose=True)
    # the transpose: <R x, y> = <x, R' y>, in 64 bits over the fp32 results
    y = randn(g, 50, 4, 128)
    a = (rope(pos, x).double() * y.double()).sum()
    b = (x.double() * rope(pos, y, transpose=True).double()).sum()
    n = (R.rotate_magnitude(x, 32, rope.value_factor, True) * y.double().abs()).sum()
    assert abs(float(a - b)) <= 2 * 4 * U * float(2 * n)


def test_rotary_gradient_by_differences():
    """d <w, R x> / dx along a direction, by central differences (the map is linear,
    so only fp32's roundings remain)."""
    g = gen(6)
    rope = RotaryEmbedding(32, scaling=RotaryScaling("yarn", 4.0, original_positions=64))
    pos = torch.arange(9, device="cuda") * 31
    x, w, d = (randn(g, 9, 3, 32) for _ in range(3))
    grad = rope(pos, w, transpose=True)
    h = 0.5
    diff = ((rope(pos, x + h * d).double() - rope(pos, x - h * d).double()) * w.double()).sum() / (2 * h)
    size = (R.rotate_magnitude(x, 16, rope.value_factor, False)
            + R.rotate_magnitude(d, 16, rope.value_factor, False)) * w.double().abs()
    assert abs(float(diff - (grad.double() * d.double()).sum())) <= 16 * U * float(size.sum())


def test_rotary_far_and_negative_positions():
    g = gen(7)
    rope = RotaryEmbedding(64, layout="half")
    x = randn(g, 6, 2, 64)
    pos = torch.tensor([0, -1, -100000, 1 << 20, (1 << 31) + 12345, -(1 << 33)], device="cuda")
    check_rotated(rope(pos, x), x, pos, rope)
    assert torch.equal(rope(pos, x)[0], x[0])  # position 0 turns nothing


def test_rotary_empty_and_non_finite():
    rope = RotaryEmbedding(64, rotary_dim=32)
    none = torch.zeros(0, 4, 64, device="cuda")
    assert rope(torch.zeros(0, dtype=torch.int64, device="cuda"), none).shape == (0, 4, 64)
    x = torch.ones(2, 2, 64, device="cuda", dtype=BF16)
    x[0, 0, 3] = math.nan
    x[0, 1, 40] = math.inf
    y = rope(torch.tensor([3, 4], device="cuda"), x)
    bad = ~torch.isfinite(y)
    assert bad[0, 0, 3] and bad[0, 0, 19] and int(bad.sum()) == 3 and y[0, 1, 40] == math.inf


def test_rotary_refusals():
    rope = RotaryEmbedding(64)
    x = torch.zeros(4, 2, 64, device="cuda")
    p = torch.arange(4, device="cuda")
    for args, kind in (((p, x[..., :32]), ValueError), ((p[:3], x), ValueError), ((p.float(), x), TypeError),
                       ((p.cpu(), x), ValueError), ((p, x.double()), TypeError), ((p, x[0]), ValueError),
                       ((p, x, x.half()), ValueError), ((p, x, x[:3]), ValueError),
                       ((p[None], x), ValueError)):
        with pytest.raises(kind):
            rope(*args)
    with pytest.raises(ValueError):
        rope(p, x[:1].expand(4, 2, 64), inplace=True)
    with pytest.raises(ValueError):
        rope(p, torch.zeros(4, 64, 2, device="cuda").transpose(1, 2), inplace=True)
    with pytest.raises(ValueError):
        RotaryEmbedding(64, device="cpu")(p, x)
    with pytest.raises(ValueError):
        rope(p, x, x, inplace=True)


def test_copies_have_tensors_of_their_own():
    """copy.deepcopy and pickle rebuild what the calls hand to the library."""
    g = gen(9)
    x = randn(g, 5, 2, 64, dtype=BF16)
    p = torch.arange(5, device="cuda")
    rope, pool = RotaryEmbedding(64), KVPagePool(2, 2, 64, page_size=4)
    pool.write(x, x, p)
    want = rope(p, x), pool.read(p)
    for make in (copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))):
        r, q = make(rope), make(pool)
        assert r.turns.data_ptr() != rope.turns.data_ptr() and q.k.data_ptr() != pool.k.data_ptr()
        assert torch.equal(r(p, x), want[0]) and torch.equal(q.read(p)[0], want[1][0])
        q.write(-x, x, p)
        assert torch.equal(pool.read(p)[0], want[1][0]) and not torch.equal(q.read(p)[0], want[1][0])
        with pytest.raises(AttributeError):
            r.turns = None
        with pytest.raises(AttributeError):
            q.k = None


# --------------------------------------------------------------------- pool
SHAPES = [(8, 128, 16), (3, 64, 16), (2, 80, 16), (2, 80, 80), (1, 45, 16), (5, 96, 32), (2, 256, 64),
          (2, 512, 16), (3, 24, 12), (2, 8, 8)]


def fill(pool, byte=0x5A):
    """Every byte of the pool set, so that untouched rows can be told."""
    for t in (pool.k, pool.v, pool.scale_k, pool.scale_v):
        if t is not None:
            t.view(torch.uint8).fill_(byte)


def snapshot(pool):
    return [None if t is None else t.clone() for t in (pool.k, pool.v, pool.scale_k, pool.scale_v)]


def expect_rows(pool, before, k, v, slots):
    """The pool's tensors after a write: the oracle's rows in their slots."""
    P = pool.page_size
    for j, x in enumerate((k, v)):
        payload, scales = R.encode(x.cpu(), pool.precision, pool.int4_group_size)
        for got, old, rows in ((pool.k, pool.v)[j], before[j], payload), \
                ((pool.scale_k, pool.scale_v)[j], before[2 + j], scales):
            if got is None:
                continue
            want = old.cpu()
            for t, s in enumerate(slots.tolist()):
                if 0 <= s < pool.num_slots:
                    want[s // P, :, s % P] = rows[t]
            assert np.array_equal(bits(got), bits(want))


@pytest.mark.parametrize("precision", ["fp32", "fp16", "int8", "int4"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H,D,group", SHAPES)
def test_pool_write_and_read(precision, dtype, H, D, group):
    g = gen(H * 1000 + D)
    pool = KVPagePool(9, H, D, page_size=7, precision=precision, dtype=dtype, int4_group_size=group)
    fill(pool)
    T = 41
    k, v = randn(g, T, H, D, dtype=dtype, scale=3.0), randn(g, T, H, D, dtype=dtype)
    k[5] = 0
    slots = torch.randperm(63, generator=g, device="cuda")[:T]
    slots[::6] = -1
    slots[1], slots[2] = 63, 1 << 40   # outside the pool
    before = snapshot(pool)
    pool.write(k, v, slots)
    expect_rows(pool, before, k, v, slots)
    inside = (slots >= 0) & (slots < 63)
    for out in (F32, dtype, F16):
        gk, gv = pool.read(slots, dtype=out)
        for got, x in ((gk, k), (gv, v)):
            payload, scales = R.encode(x, precision, pool.int4_group_size)
            want = R.decode(payload, scales, precision, D)
            # one product of fp32 rounding, then the output's
            want = torch.where(inside[:, None, None], want, torch.zeros_like(want)).float().to(out)
            assert got.dtype == out and torch.equal(got, want)


@pytest.mark.parametrize("precision", ["fp32", "int8", "int4"])
def test_pool_rows_are_the_stores(precision):
    """A pool's rows are PagedKVStore's, bit for bit."""
    g = gen(3)
    H, D, P, T = 4, 64, 8, 21
    k, v = randn(g, 1, H, T, D, dtype=BF16), randn(g, 1, H, T, D, dtype=BF16)
    store = PagedKVStore(1, H, D, page_size=P, device="cuda")
    store.append(k, v, precision)
    pool = KVPagePool(3, H, D, page_size=P, precision=precision)
    pool.write(k[0].transpose(0, 1), v[0].transpose(0, 1), torch.arange(T, device="cuda"))
    for i, page in enumerate(store._live()):
        n = page.num_tokens
        for name in ("k", "v", "scale_k", "scale_v"):
            mine, theirs = getattr(pool, name), getattr(page, name)
            assert (mine is None) == (theirs is None)
            if mine is not None:
                assert np.array_equal(bits(mine[i, :, :n]), bits(theirs[0].reshape(mine[i, :, :n].shape)))
    gk, gv = pool.read(torch.arange(T, device="cuda"))
    sk, sv = store.gather()
    assert torch.equal(gk.transpose(0, 1), sk[0]) and torch.equal(gv.transpose(0, 1), sv[0])


def test_pool_strides_and_alignment():
    g = gen(4)
    H, D, T = 4, 64, 19
    x = randn(g, T, 3 * H * D, dtype=BF16)
    k, v = x[:, H * D:2 * H * D].unflatten(1, (H, D)), x[:, 2 * H * D:].unflatten(1, (H, D))
    slots = torch.arange(T, device="cuda") * 2
    want = KVPagePool(5, H, D, page_size=8)
    want.write(k.contiguous(), v.contiguous(), slots)
    flat = torch.empty(T * H * D + 1, dtype=BF16, device="cuda")
    odd = flat[1:].view(T, H, D)
    odd.copy_(k)
    heads_first = k.transpose(0, 1).contiguous().transpose(0, 1)
    last = k.transpose(1, 2).contiguous().transpose(1, 2)
    for kk in (k, odd, heads_first, last):
        pool = KVPagePool(5, H, D, page_size=8)
        pool.write(kk, v, torch.arange(2 * T, device="cuda")[::2])
        for name in ("k", "v", "scale_k", "scale_v"):
            assert np.array_equal(bits(getattr(pool, name)), bits(getattr(want, name)))


@pytest.mark.parametrize("precision", ["fp32", "int8", "int4"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D,rot", [(128, 128), (64, 32), (80, 20), (45, 6)])
def test_pool_rotated_write(precision, dtype, layout, D, rot):
    """Rotating on the way gives the bytes of rotating first."""
    g = gen(D + rot)
    H, T = 3, 50
    rope = RotaryEmbedding(D, rotary_dim=rot, layout=layout,
                           scaling=RotaryScaling("yarn", 2.0, original_positions=64))
    k, v = randn(g, T, H, D, dtype=dtype), randn(g, T, H, D, dtype=dtype)
    pos = torch.randint(0, 100000, (2 * T,), generator=g, device="cuda")[::2]
    slots = torch.randperm(T + 6, generator=g, device="cuda")[:T]
    slots[7] = -1
    a, b = (KVPagePool(8, H, D, page_size=7, precision=precision, dtype=dtype) for _ in range(2))
    a.write(k, v, slots, rotary=rope, positions=pos.int() if T % 2 else pos)
    b.write(rope(pos, k), v, slots)
    for name in ("k", "v", "scale_k", "scale_v"):
        if getattr(a, name) is not None:
            assert np.array_equal(bits(getattr(a, name)), bits(getattr(b, name)))


def test_pool_non_finite_rows():
    """A NaN makes its int8 row (int4 group) NaN, and no other."""
    for precision, width in (("int8", 64), ("int4", 16)):
        for dtype in (F32, F16, BF16):
            pool = KVPagePool(2, 2, 64, page_size=4, precision=precision, dtype=dtype)
            k = torch.ones(2, 2, 64, device="cuda", dtype=dtype)
            k[1, 0, 20] = math.nan
            pool.write(k, k, torch.tensor([1, 6], device="cuda"))
            gk, _ = pool.read(torch.tensor([1, 6], device="cuda"))
            bad = torch.isnan(gk)
            assert int(bad.sum()) == width and bad[1, 0, 20]


def test_pool_empty_calls_and_refusals():
    pool = KVPagePool(4, 2, 64)
    x = torch.zeros(3, 2, 64, device="cuda", dtype=BF16)
    s = torch.arange(3, device="cuda")
    before = snapshot(pool)
    pool.write(x[:0], x[:0], s[:0])
    assert all(a is None or torch.equal(a, b) for a, b in zip(before, snapshot(pool)))
    k, v = pool.read(s[:0])
    assert k.shape == (0, 2, 64)
    rope = RotaryEmbedding(64)
    for args, kw, kind in (((x.float(), x, s), {}, TypeError), ((x, x[:2], s), {}, ValueError),
                           ((x[:, :1], x[:, :1], s), {}, ValueError), ((x, x, s[:2]), {}, ValueError),
                           ((x, x, s.int()), {}, TypeError), ((x, x, s.cpu()), {}, ValueError),
                           ((x, x, s[None]), {}, ValueError), ((x, x, s), {"rotary": rope}, ValueError),
                           ((x, x, s), {"positions": s}, ValueError),
                           ((x, x, s), {"rotary": RotaryEmbedding(32), "positions": s}, ValueError),
                           ((x, x, s), {"rotary": rope, "positions": s[:2]}, ValueError)):
        with pytest.raises(kind):
            pool.write(*args, **kw)
    with pytest.raises(TypeError):
        pool.read(s, dtype=torch.int8)
    with pytest.raises(TypeError):
        pool.read(s.int())
    with pytest.raises(ValueError):
        pool.read(s.cpu())


def test_pool_past_32_bit_offsets():
    """Rows beyond 4 GiB of a tensor: written, read and attended to."""
    pool = KVPagePool(1 << 16, 8, 128, page_size=40, precision="fp32", dtype=BF16)
    assert pool.k.numel() * 2 > 1 << 32
    g = gen(8)
    k, v = randn(g, 80, 8, 128, dtype=BF16), randn(g, 80, 8, 128, dtype=BF16)
    top = pool.num_slots
    slots = torch.cat((torch.arange(top - 40, top, device="cuda"), torch.arange(40, device="cuda")))
    pool.write(k, v, slots)
    gk, gv = pool.read(slots, dtype=BF16)
    assert torch.equal(gk, k) and torch.equal(gv, v)
    assert torch.equal(pool.k[-1].transpose(0, 1), k[:40])
    q = randn(g, 1, 16, 128, dtype=BF16)
    table = torch.tensor([[(1 << 16) - 1, 0]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([77], dtype=torch.int32, device="cuda")
    small = KVPagePool(2, 8, 128, page_size=40, precision="fp32", dtype=BF16)
    small.write(k, v, torch.arange(80, device="cuda"))
    two = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    assert torch.equal(paged_attention(q, pool, table, lens), paged_attention(q, small, two, lens))


# ---------------------------------------------------------------- attention
def make_cache(g, lens, H, D, P, precision, dtype, group=16, extra=3, width=None):
    """A pool whose pages hold sequences of ``lens`` in no order, NaN (or NaN scales)
    wherever no position is."""
    need = [(n + P - 1) // P for n in lens]
    pages = sum(need) + extra
    pool = KVPagePool(pages, H, D, page_size=P, precision=precision, dtype=dtype, int4_group_size=group)
    for t in (pool.k, pool.v, pool.scale_k, pool.scale_v):
        if t is not None:
            t.fill_(math.nan if t.is_floating_point() else 0x7B)
    free = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width or max(1, max(need))), -1, dtype=torch.int32, device="cuda")
    slots, at = [], 0
    for b, n in enumerate(lens):
        mine = free[at:at + need[b]]
        table[b, :need[b]] = mine
        at += need[b]
        t = torch.arange(n, device="cuda")
        slots.append(mine.long()[t // P] * P + t % P)
    slots = torch.cat(slots)
    k = randn(g, slots.numel(), H, D, dtype=dtype)
    v = randn(g, slots.numel(), H, D, dtype=dtype)
    k[..., 3 % D] *= 6
    pool.write(k, v, slots)
    return pool, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def check_attention(q, pool, table, lengths, window=None, sm_scale=None):
    """Against the oracle, twice: with the table as it is, and with columns of missing pages behind it
    that let the call expect long sequences (whose tiles are dealt to workgroups and joined)."""
    P = pool.page_size
    more = torch.full((table.shape[0], -(-3200 // P)), -1, dtype=torch.int32, device=table.device)
    scale = 1 / math.sqrt(pool.head_dim) if sm_scale is None else sm_scale
    want, wlse, weight, reach, peak = R.attend(q, R.pool_values(pool, "k"), R.pool_values(pool, "v"), table, lengths,
                                               scale, window)
    n = min(int(lengths.max()), table.shape[1] * P) if lengths.numel() else 0
    slip = (pool.head_dim + 16) * U * (1 + reach)        # a score's error
    part = 2.0 ** -16 if q.dtype != F32 else 0.0
    rel = (2 * slip + (n / 4 + 64) * U + part)[..., None]
    # A weight p_t s_t (s_t: the factor of a quantized row, 1 of another) in two fp16 parts is
    # scaled so that the largest of a row is 2^14 (2^13 at least where the scale is no power of two);
    # fp16 steps by 2^-24 there, so each is off by 2^-25 at most, 2^-38 of the largest. Times the
    # row's |v_td| / s_t, at most 128 for int8 and int4: 2^-38 n max_t(s_t p_t) 128, and s_t <= max |v_t|;
    # for 16-bit rows 2^-38 n max_t(p_t) max |v|. It shows where the heaviest rows have a 0.
    floor = 2.0 ** -38 * n * peak[..., None] if q.dtype != F32 else 0.0
    tol = rel * weight + floor
    tol = tol + HALF_STEP[q.dtype] * (want.abs() + tol) + TINY[q.dtype]
    for tab in (table, torch.cat((table, more), 1)):
        out, lse = paged_attention(q, pool, tab, lengths, sm_scale=sm_scale, window=window, return_lse=True)
        again = paged_attention(q, pool, tab, lengths, sm_scale=sm_scale, window=window)
        assert np.array_equal(bits(again), bits(out))
        assert out.dtype == q.dtype and out.shape == q.shape and lse.dtype == F32
        nan = torch.isnan(want)  # a visible row may hold one
        assert torch.equal(torch.isnan(out), nan)
        off = ((out.double() - want).abs() / tol)[~nan]
        assert (off <= 1).all(), float(off.max())
        nan = torch.isnan(wlse)
        assert torch.equal(torch.isnan(lse), nan)
        empty = torch.isneginf(wlse)
        assert torch.equal(torch.isneginf(lse), empty) and (out[empty] == 0).all()
        live = ~(empty | nan)
        off = (lse.double() - wlse).abs()[live]
        assert (off <= (slip + (n / 4 + 64) * U + 4 * U * wlse.abs())[live]).all()
        if window is not None and lengths.numel() and int(lengths.max()) > table.shape[1] * P:
            break  # the positions that are cut would be in the window
    return out


@pytest.mark.parametrize("precision", ["fp32", "fp16", "int8", "int4"])
@pytest.mark.parametrize("qt,dtype", [(BF16, BF16), (F16, F16), (F32, F32), (F16, BF16), (BF16, F32),
                                      (F32, BF16), (BF16, F16), (F16, F32)])
@pytest.mark.parametrize("D", [64, 128, 80])
def test_attention_types(precision, qt, dtype, D):
    g = gen(D)
    lens = [1, 300, 0, 33, 129, 64]
    pool, table, lengths = make_cache(g, lens, 2, D, 16, precision, dtype)
    check_attention(randn(g, len(lens), 8, D, dtype=qt), pool, table, lengths)


@pytest.mark.parametrize("P", [1, 3, 8, 16, 24, 32, 64, 200])
@pytest.mark.parametrize("precision", ["fp32", "int8", "int4"])
def test_attention_page_sizes(P, precision):
    g = gen(P)
    lens = [2 * P, 2 * P + 1, max(1, 2 * P - 1), 257, 31, 1]
    pool, table, lengths = make_cache(g, lens, 3, 64, P, precision, BF16)
    check_attention(randn(g, len(lens), 3, 64, dtype=BF16), pool, table, lengths)


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (7, 7), (12, 4), (8, 1), (16, 1), (17, 1), (40, 1), (64, 2)])
@pytest.mark.parametrize("n", [1, 100, 700])
@pytest.mark.parametrize("precision", ["fp32", "int8"])
def test_attention_groups(Hq, Hk, n, precision):
    """Groups of one to more query heads than a tile holds."""
    g = gen(Hq * 10 + Hk)
    pool, table, lengths = make_cache(g, [n, n // 2], Hk, 128, 32, precision, BF16)
    check_attention(randn(g, 2, Hq, 128, dtype=BF16), pool, table, lengths)


@pytest.mark.parametrize("D,group", [(8, 8), (16, 16), (24, 8), (40, 8), (72, 24), (96, 32), (104, 104), (112, 16),
                                     (120, 40), (128, 64), (33, 16), (45, 9), (100, 4), (160, 16), (256, 16),
                                     (512, 64), (3, 16)])
@pytest.mark.parametrize("precision", ["fp32", "int8", "int4"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_head_sizes(D, group, precision, dtype):
    g = gen(D)
    pool, table, lengths = make_cache(g, [150, 5, 0, 260], 2, D, 16, precision, dtype, group=group)
    check_attention(randn(g, 4, 4, D, dtype=dtype), pool, table, lengths)


@pytest.mark.parametrize("window", [1, 31, 32, 100, 128, 129, 1000, 5000])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_window(window, dtype):
    g = gen(window)
    lens = [1, 32, 100, 127, 129, 1500, 0]
    pool, table, lengths = make_cache(g, lens, 2, 64, 24, "int8", dtype)
    check_attention(randn(g, len(lens), 6, 64, dtype=dtype), pool, table, lengths, window=window)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens", [[20000], [9000, 1, 0, 300, 4096, 17], [0, 0], [513] * 40])
def test_attention_long_and_uneven(lens, dtype):
    """Items over many workgroups, workgroups over many items."""
    g = gen(sum(lens) + 1)
    pool, table, lengths = make_cache(g, lens, 2, 64, 32, "int8", dtype)
    check_attention(randn(g, len(lens), 4, 64, dtype=dtype), pool, table, lengths)


@pytest.mark.parametrize("precision,dtype", [("fp32", BF16), ("fp32", F16), ("fp32", F32), ("int8", BF16), ("int4", BF16),
                                             ("int4", F16)])
@pytest.mark.parametrize("D,P", [(64, 8), (128, 24), (80, 16), (128, 10)])
def test_attention_many_items(precision, dtype, D, P):
    """More items than the chip has CUs."""
    g = gen(24)
    lens = torch.randint(0, 100, (90,), generator=torch.Generator().manual_seed(7)).tolist()
    lens[5] = 300
    pool, table, lengths = make_cache(g, lens, 3, D, P, precision, dtype)
    check_attention(randn(g, 90, 6, D, dtype=dtype), pool, table, lengths)


@pytest.mark.parametrize("longest", [900, 3300])
def test_attention_many_sequences(longest):
    """More sequences than a block has threads."""
    g = gen(11)
    lens = torch.randint(0, 60, (700,), generator=torch.Generator().manual_seed(131)).tolist()
    lens[3], lens[650] = longest, 450
    pool, table, lengths = make_cache(g, lens, 1, 64, 16, "int8", BF16)
    check_attention(randn(g, 700, 2, 64, dtype=BF16), pool, table, lengths)


@pytest.mark.parametrize("precision", ["fp32", "int8", "int4"])
@pytest.mark.parametrize("D", [64, 45])
def test_attention_missing_pages_and_odd_lengths(precision, D):
    """Pages outside the pool take no part, wherever they are; lengths past the table
    are cut, negative ones empty."""
    g = gen(12)
    lens = [300, 300, 300, 300, 50, 50]
    pool, table, lengths = make_cache(g, lens, 2, D, 16, precision, BF16)
    table[0, 0] = -1
    table[1, 3:15] = -1
    table[2, :] = -1
    table[3, 5], table[3, 6], table[3, 7] = pool.num_pages, 2 ** 31 - 1, -(2 ** 31)
    table[4, 4:] = -7
    lengths[4] = 10000       # past the table: its pages there are missing
    lengths[5] = -5
    check_attention(randn(g, 6, 4, D, dtype=BF16), pool, table, lengths)
    short = table[:, :2]     # a strided table that ends before the lengths do
    check_attention(randn(g, 6, 4, D, dtype=BF16), pool, short, lengths)
    none = table[:, :0]
    q = randn(g, 6, 4, D, dtype=BF16)
    out, lse = paged_attention(q, pool, none, lengths, return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()


def test_attention_shared_pages():
    """Sequences that share a prefix share its pages."""
    g = gen(13)
    pool, table, lengths = make_cache(g, [200, 190], 2, 128, 16, "int4", BF16)
    table[1, :8] = table[0, :8]
    check_attention(randn(g, 2, 4, 128, dtype=BF16), pool, table, lengths)


@pytest.mark.parametrize("qt,dtype,precision", [(BF16, BF16, "fp32"), (BF16, BF16, "int8"), (F16, F16, "fp32"),
                                                (F16, F16, "int8"), (F16, F16, "int4"), (BF16, BF16, "int4"),
                                                (F32, F32, "fp32"), (F32, F32, "int8"), (BF16, F32, "int4")])
@pytest.mark.parametrize("qs,ks,vs", [(30.0, 1.0, 1.0), (1e-4, 1e-4, 1e-4), (1.0, 100.0, 1e-3), (100.0, 1e-2, 100.0),
                                      (1.0, 1.0, 3000.0)])
def test_attention_scales(qt, dtype, precision, qs, ks, vs):
    """Peaked and flat rows, and values from 1e-4 to 1e4."""
    g = gen(14)
    D, lens = 128, [400, 77]
    pool, table, lengths = make_cache(g, lens, 2, D, 16, precision, dtype)
    slots = torch.arange(pool.num_slots, device="cuda")
    k = randn(g, pool.num_slots, 2, D, dtype=dtype, scale=ks)
    v = randn(g, pool.num_slots, 2, D, dtype=dtype, scale=vs)
    # scales that differ from row to row
    v *= torch.logspace(-2, 0, pool.num_slots, device="cuda")[:, None, None].to(dtype)
    pool.write(k, v, slots)
    check_attention(randn(g, 2, 8, D, dtype=qt, scale=qs), pool, table, lengths)


@pytest.mark.parametrize("dtype,precision,size", [(BF16, "fp32", 2.0 ** 126), (F32, "fp32", 2.0 ** 126),
                                                  (BF16, "int8", 2.0 ** 126), (F16, "fp32", 32768.0),
                                                  (BF16, "int4", 2.0 ** 126), (BF16, "fp32", 2.0 ** -100),
                                                  (BF16, "int8", 2.0 ** -70), (BF16, "int4", 2.0 ** -70)])
@pytest.mark.parametrize("D", [64, 45])
def test_attention_values_at_the_range_ends(dtype, precision, size, D):
    """Values near the type's largest and down to 2^-100 come out finite and as exact as others."""
    g = gen(25)
    pool, table, lengths = make_cache(g, [70, 300], 1, D, 16, precision, dtype)
    slots = torch.arange(pool.num_slots, device="cuda")
    k = randn(g, pool.num_slots, 1, D, dtype=dtype)
    v = (torch.rand(pool.num_slots, 1, D, generator=g, device="cuda") * 2 - 1) * size
    pool.write(k, v.to(dtype), slots)
    out = check_attention(randn(g, 2, 4, D, dtype=dtype), pool, table, lengths)
    assert torch.isfinite(out).all() and (out != 0).any()


@pytest.mark.parametrize("precision", ["fp32", "int8"])
def test_attention_extreme_rows(precision):
    """Rows whose scales lie 2^60 apart, a row of zeros, equal rows, and a q of zeros."""
    g = gen(15)
    pool, table, lengths = make_cache(g, [300], 1, 64, 32, precision, BF16)
    k, v = randn(g, 300, 1, 64, dtype=BF16), randn(g, 300, 1, 64, dtype=BF16)
    v[100:200] *= 2.0 ** 30
    v[200:] *= 2.0 ** -30
    k[100:200] *= -1
    v[7], k[7] = 0, 0
    k[20:30] = k[20]
    t = torch.arange(300, device="cuda")
    pool.write(k, v, table[0].long()[t // 32] * 32 + t % 32)
    q = randn(g, 1, 4, 64, dtype=BF16)
    q[0, 1] = 0
    q[0, 2] *= 2.0 ** -60
    check_attention(q, pool, table, lengths)


@pytest.mark.parametrize("precision", ["fp32", "int8", "int4"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_nan_in_a_visible_row(precision, dtype):
    """A NaN key or value in a row that takes part makes its heads NaN, and only those."""
    g = gen(16)
    for name in ("k", "v"):
        pool, table, lengths = make_cache(g, [140, 140], 2, 64, 16, precision, dtype)
        page = int(table[0, 4])
        row = getattr(pool, name) if precision == "fp32" else getattr(pool, "scale_" + name)
        row[page, 1, 3] = math.nan
        q = randn(g, 2, 4, 64, dtype=dtype)
        out, lse = paged_attention(q, pool, table, lengths, return_lse=True)
        assert torch.isnan(out[0, 2:]).all() and torch.isfinite(out[0, :2]).all()
        assert torch.isfinite(out[1]).all()
        assert torch.isnan(lse[0, 2:]).all() == (name == "k")
        # the same row behind the sequence's end does nothing
        lengths[0] = 4 * 16 + 3
        assert torch.isfinite(paged_attention(q, pool, table, lengths)).all()


@pytest.mark.parametrize("qt,dtype,precision,part", [(F16, F16, "fp32", 2.0 ** -21), (BF16, BF16, "int8", 2.0 ** -21),
                                                     (BF16, F32, "int8", 2.0 ** -21), (BF16, BF16, "int4", 2.0 ** -21),
                                                     (F16, F16, "int4", 2.0 ** -19), (BF16, BF16, "fp32", 2.0 ** -15)])
def test_attention_weights_keep_both_parts(qt, dtype, precision, part):
    """Two-part weights are 2^-22 (fp16) or 2^-16 (bf16) exact for every single one of many: where a row's
    values cancel, a weight that lost its low part (2^-12) would show. (int4 with fp16 scales: its
    scales are in two parts as well, 2^-20.)"""
    g = gen(23)
    B, n, H, D = 6000, 6, 2, 64
    pool = KVPagePool(B, 1, D, page_size=8, precision=precision, dtype=dtype)
    k, v = randn(g, B * n, 1, D, dtype=dtype), randn(g, B * n, 1, D, dtype=dtype)
    at = torch.arange(B * n, device="cuda")
    pool.write(k, v, at // n * 8 + at % n)
    q = randn(g, B, H, D, dtype=qt)
    table = torch.arange(B, dtype=torch.int32, device="cuda")[:, None]
    out = paged_attention(q, pool, table, torch.full((B,), n, dtype=torch.int32, device="cuda")).double()
    kk, vv = (R.pool_values(pool, x)[:, 0, :n] for x in ("k", "v"))          # [B, n, D]
    s = torch.matmul(q.double(), kk.transpose(1, 2).contiguous()) / math.sqrt(D)
    p = torch.softmax(s, -1)
    want, weight = torch.matmul(p, vv), torch.matmul(p, vv.abs())
    slip = (D + 16) * U * (1 + s.abs().amax(-1, keepdim=True) * 8)
    tol = (2 * slip + 80 * U + part) * weight
    tol = tol + HALF_STEP[qt] * (want.abs() + tol) + TINY[qt]
    assert ((out - want).abs() <= tol).all(), float(((out - want).abs() / tol).max())


def test_attention_strides_and_scale():
    g = gen(17)
    pool, table, lengths = make_cache(g, [130, 60, 7], 2, 64, 16, "int8", BF16)
    x = randn(g, 3, 3 * 8 * 64, dtype=BF16)
    q = x[:, 8 * 64:16 * 64].unflatten(1, (8, 64))
    want = check_attention(q, pool, table, lengths, sm_scale=0.3)
    flat = torch.empty(3 * 8 * 64 + 1, dtype=BF16, device="cuda")
    odd = flat[1:].view(3, 8, 64)
    odd.copy_(q)
    wide = torch.full((3, 40), 2 ** 30, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    lens2 = torch.stack((lengths, lengths), 1)[:, 0]
    for qq in (odd, q.transpose(0, 1).contiguous().transpose(0, 1), q.transpose(1, 2).contiguous().transpose(1, 2)):
        assert torch.equal(paged_attention(qq, pool, wide[:, :table.shape[1]], lens2, sm_scale=0.3), want)
    check_attention(q, pool, table, lengths, sm_scale=-0.1)
    check_attention(q, pool, table, lengths, sm_scale=0.0)


def test_attention_deterministic():
    g = gen(18)
    pool, table, lengths = make_cache(g, [5000, 3, 2000], 2, 128, 16, "int4", BF16)
    q = randn(g, 3, 8, 128, dtype=BF16)
    first = paged_attention(q, pool, table, lengths)
    for _ in range(5):
        assert torch.equal(paged_attention(q, pool, table, lengths), first)


def test_attention_refusals():
    pool = KVPagePool(4, 2, 64)
    q = torch.zeros(3, 4, 64, device="cuda", dtype=BF16)
    t = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    n = torch.ones(3, dtype=torch.int32, device="cuda")
    for args, kw, kind in (((q[..., :32], pool, t, n), {}, ValueError), ((q[:, :3], pool, t, n), {}, ValueError),
                           ((q[:, :0], pool, t, n), {}, ValueError), ((q.double(), pool, t, n), {}, TypeError),
                           ((q, pool, t.long(), n), {}, TypeError), ((q, pool, t, n.long()), {}, TypeError),
                           ((q, pool, t[:2], n), {}, ValueError), ((q, pool, t, n[:2]), {}, ValueError),
                           ((q, pool, t.cpu(), n), {}, ValueError), ((q, pool, t, n.cpu()), {}, ValueError),
                           ((q[0], pool, t, n), {}, ValueError), ((q, pool, t, n), {"window": 0}, ValueError),
                           ((q, pool, t, n), {"window": -3}, ValueError),
                           ((q, KVPagePool(4, 2, 64, device="cpu"), t, n), {}, ValueError)):
        with pytest.raises(kind):
            paged_attention(*args, **kw)
    none = paged_attention(q[:0], pool, t[:0], n[:0])
    assert none.shape == (0, 4, 64)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("precision,dtype", [("int8", BF16), ("int4", BF16), ("fp32", F16), ("fp32", F32)])
def test_decode_loop(precision, dtype):
    """Two prompts of different lengths written with their keys rotated, then steps of one
    token: rotate the query, write the key, attend."""
    g = gen(20)
    B, Hq, Hk, D, P, steps = 2, 8, 2, 64, 8, 12
    rope = RotaryEmbedding(D, layout="interleaved", scaling=RotaryScaling("linear", 2.0))
    pool = KVPagePool(24, Hk, D, page_size=P, precision=precision, dtype=dtype)
    table = torch.randperm(24, generator=g, device="cuda")[:16].view(2, 8).to(torch.int32)
    prompt = [37, 5]
    ks, vs = [[], []], [[], []]

    def slots_of(b, t):
        return table[b].long()[t // P] * P + t % P

    def append(b, k, v, first):
        t = torch.arange(first, first + k.shape[0], device="cuda")
        ks[b].append(rope(t, k))
        vs[b].append(v)
        return t

    for b, n in enumerate(prompt):
        k, v = randn(g, n, Hk, D, dtype=dtype), randn(g, n, Hk, D, dtype=dtype)
        t = append(b, k, v, 0)
        pool.write(k, v, slots_of(b, t), rotary=rope, positions=t)
    for s in range(steps):
        pos = torch.tensor([prompt[0] + s, prompt[1] + s], device="cuda")
        x = randn(g, B, (Hq + 2 * Hk) * D, dtype=dtype)
        q, k, v = (y.unflatten(1, (-1, D)) for y in x.split((Hq * D, Hk * D, Hk * D), 1))
        slots = torch.stack([slots_of(b, pos[b]) for b in range(B)])
        pool.write(k, v, slots, rotary=rope, positions=pos)
        for b in range(B):
            append(b, k[b:b + 1], v[b:b + 1], prompt[b] + s)
        lengths = (pos + 1).int()
        out = check_attention(rope(pos, q), pool, table, lengths)
    # and the pool holds the rows that the parts gave
    for b in range(B):
        k, v = torch.cat(ks[b]), torch.cat(vs[b])
        t = torch.arange(k.shape[0], device="cuda")
        gk, gv = pool.read(slots_of(b, t))
        for got, x in ((gk, k), (gv, v)):
            payload, scales = R.encode(x, precision, 16)
            assert torch.equal(got, R.decode(payload, scales, precision, D).float())
    assert torch.isfinite(out).all()


def step(rope, pool, pos, q, k, v, slots, table, lengths):
    """One decode step as a program runs it."""
    pool.write(k, v, slots, rotary=rope, positions=pos)
    return paged_attention(rope(pos, q), pool, table, lengths)


def test_captured_steps_replay_with_new_inputs():
    """Two captured graphs of different sizes over one pool, replayed in turn with other
    positions, slots and lengths, eager work between: every replay the eager bits."""
    g = gen(21)
    Hq, Hk, D, P = 8, 2, 128, 16
    rope = RotaryEmbedding(D)
    pools = [KVPagePool(200, Hk, D, page_size=P, precision="int8") for _ in range(2)]
    graphs = []
    for B, width in ((3, 40), (2, 6)):
        table = torch.randperm(200, generator=g, device="cuda")[:B * width].view(B, width).to(torch.int32)
        st = dict(pos=torch.zeros(B, dtype=torch.int64, device="cuda"), q=torch.zeros(B, Hq, D, dtype=BF16, device="cuda"),
                  k=torch.zeros(B, Hk, D, dtype=BF16, device="cuda"), v=torch.zeros(B, Hk, D, dtype=BF16, device="cuda"),
                  slots=torch.zeros(B, dtype=torch.int64, device="cuda"), table=table,
                  lengths=torch.ones(B, dtype=torch.int32, device="cuda"))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(rope, pools[0], **st)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(rope, pools[0], **st)
        graphs.append((graph, st, out, B, width))
    for p in pools:  # the same rows in both
        kk = randn(gen(99), p.num_slots, Hk, D, dtype=BF16)
        p.write(kk, kk, torch.arange(p.num_slots, device="cuda"))
    for i in range(6):
        for graph, st, out, B, width in graphs:
            n = torch.randint(1, width * P, (B,), generator=g, device="cuda")
            st["pos"].copy_(n - 1)
            st["lengths"].copy_(n.int())
            st["slots"].copy_(st["table"].gather(1, ((n - 1) // P)[:, None])[:, 0].long() * P + (n - 1) % P)
            for name in ("q", "k", "v"):
                st[name].copy_(randn(g, *st[name].shape, dtype=BF16))
            graph.replay()
            eager = step(rope, pools[1], **st)
            torch.cuda.synchronize()
            assert torch.equal(out, eager), i
            assert torch.equal(pools[0].k, pools[1].k) and torch.equal(pools[0].scale_v, pools[1].scale_v)


def test_two_streams_at_once():
    """Calls on two streams over one pool do not share state."""
    g = gen(22)
    pool, table, lengths = make_cache(g, [4000, 900], 2, 128, 16, "int8", BF16)
    qs = [randn(g, 2, 8, 128, dtype=BF16) for _ in range(2)]
    want = [paged_attention(q, pool, table, lengths) for q in qs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged_attention(qs[i], pool, table, lengths))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])
