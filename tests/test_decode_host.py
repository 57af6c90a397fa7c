"""Host side of the decode operators: the placing and dealing functions (run
natively), rotary scalings, refusals, and known answers of the oracle."""

import ctypes
import math
import os
import struct
import subprocess

import numpy as np
import pytest
import torch

from helpers import DT, to_np
from oracle import decode_ref as R
from oracle import oracle as O
from shadowinfer_amd import KVPagePool, RotaryEmbedding, RotaryScaling, _native, paged_attention

HERE = os.path.dirname(os.path.abspath(__file__))


def test_rows_spans_and_dealing_are_in_bounds(tmp_path):
    exe = tmp_path / "pool_index_check"
    subprocess.check_call(["gcc", "-O2", "-fsanitize=address,undefined",
                           os.path.join(HERE, "native", "pool_index_check.c"), "-o", str(exe)])
    out = subprocess.run([str(exe)], stdout=subprocess.PIPE, text=True, timeout=300)
    assert out.returncode == 0, out.stdout
    assert int(out.stdout.split()[1]) > 20000


# ------------------------------------------------------------------- rotary
def test_rotary_angles_of_the_scalings():
    R_, base, s, known = 64, 10000.0, 8.0, 2048
    plain = [base ** (-2 * i / R_) for i in range(R_ // 2)]

    def angles(kind, **kw):
        r = RotaryEmbedding(128, rotary_dim=R_, base=base, device="cpu",
                            scaling=RotaryScaling(kind, s, original_positions=known, **kw))
        assert r.turns.dtype == torch.float64
        np.testing.assert_allclose(r.turns.numpy() * 2 * math.pi, r.angles, rtol=1e-15)
        return np.array(r.angles), r.value_factor

    none = RotaryEmbedding(128, rotary_dim=R_, base=base, device="cpu")
    np.testing.assert_allclose(none.angles, plain, rtol=1e-15)
    assert none.value_factor == 1.0
    a, g = angles("linear")
    np.testing.assert_allclose(a, np.array(plain) / s, rtol=1e-15)
    a, g = angles("ntk")  # the fastest pair kept, the slowest divided by the factor
    assert a[0] == 1.0 and g == 1.0
    assert a[-1] == pytest.approx(plain[-1] / s, rel=1e-12)
    a, g = angles("bands")
    for x, y in zip(plain, a):
        turns = known * x / (2 * math.pi)
        if turns >= 4:
            assert y == pytest.approx(x, rel=1e-15)
        elif turns <= 1:
            assert y == pytest.approx(x / s, rel=1e-15)
        else:
            assert x / s < y < x
    a, g = angles("yarn")
    assert g == pytest.approx(0.1 * math.log(s) + 1.0)
    for x, y in zip(plain, a):  # the ramp's edges are rounded outwards to whole pairs
        turns = known * x / (2 * math.pi)
        assert x / s * (1 - 1e-12) <= y <= x * (1 + 1e-12)
        if turns >= 32 * base ** (2 / R_):
            assert y == pytest.approx(x, rel=1e-12)
        if turns <= base ** (-2 / R_):
            assert y == pytest.approx(x / s, rel=1e-12)


@pytest.mark.parametrize("kw", [dict(head_dim=0), dict(head_dim=2000), dict(head_dim=64, rotary_dim=3),
                                dict(head_dim=64, rotary_dim=66), dict(head_dim=64, rotary_dim=0),
                                dict(head_dim=64, layout="other"), dict(head_dim=64, base=1.0),
                                dict(head_dim=64, base=float("nan"))])
def test_rotary_constructor_refuses(kw):
    with pytest.raises(ValueError):
        RotaryEmbedding(device="cpu", **kw)


def test_rotary_scaling_refuses():
    for args in (("other", 2.0), ("linear", 0.5), ("linear", float("inf")), ("yarn", 2.0, 0),
                 ("yarn", 2.0, 4096, 1.0, 1.0), ("bands", 2.0, 4096, 32.0, 1.0, 4.0, 4.0)):
        with pytest.raises(ValueError):
            RotaryScaling(*args)
    with pytest.raises(ValueError):
        RotaryEmbedding(64, rotary_dim=2, scaling=RotaryScaling("ntk", 2.0), device="cpu")


def test_pool_constructor_refuses_and_sizes():
    for kw in (dict(num_pages=0), dict(num_heads=0), dict(head_dim=0), dict(head_dim=600),
               dict(page_size=0), dict(precision="fp8"), dict(int4_group_size=0),
               dict(num_pages=1 << 20, num_heads=64, page_size=32)):
        with pytest.raises(ValueError):
            KVPagePool(**{**dict(num_pages=4, num_heads=2, head_dim=64, device="cpu"), **kw})
    with pytest.raises(TypeError):
        KVPagePool(4, 2, 64, dtype=torch.float64, device="cpu")
    p = KVPagePool(4, 2, 45, page_size=3, precision="int4", dtype=torch.float16, device="cpu")
    assert p.int4_group_size == 45 and tuple(p.k.shape) == (4, 2, 3, 23)
    assert tuple(p.scale_v.shape) == (4, 2, 3, 1) and p.scale_v.dtype == torch.float16
    assert p.num_slots == 12 and p.data_plane_bytes() == 2 * 24 * (23 + 2)
    p = KVPagePool(4, 2, 64, precision="fp32", dtype=torch.bfloat16, device="cpu")
    assert p.k.dtype == torch.bfloat16 and p.scale_k is None


def test_host_tensors_are_refused():
    pool = KVPagePool(4, 2, 64, device="cpu")
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    rope = RotaryEmbedding(64, device="cpu")
    with pytest.raises(RuntimeError):
        rope(torch.arange(3), x)
    with pytest.raises(RuntimeError):
        pool.write(x, x, torch.arange(3))
    with pytest.raises(RuntimeError):
        pool.read(torch.arange(3))
    with pytest.raises(RuntimeError):
        paged_attention(x, pool, torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32))


def test_abi_refuses_before_any_launch():
    """Bad arguments return 1 with a message; no pointer is touched."""
    lib = _native.load()
    rows = (ctypes.c_int64 * 9)(16, 16, 2, 0, 128, 64, 0, 128, 64)

    def rotation(pairs=32, freq=16):
        return ctypes.create_string_buffer(struct.pack("=qqQd", pairs, 0, freq, 1.0))

    def rotary(dtype=2, B=1, S=4, D=64, pairs=32, q=rows, freq=16, pos=16, spec=True):
        return lib.si_rotary(rotation(pairs, freq) if spec else None, q, None, dtype, B, S, D, 0, pos, 1, 0,
                             1, None)

    for kw in (dict(dtype=5), dict(D=0), dict(D=2048), dict(pairs=33), dict(pairs=0), dict(B=-1),
               dict(S=1 << 31), dict(q=None), dict(freq=0), dict(pos=None), dict(spec=False)):
        assert rotary(**kw) == 1 and b"si_rotary" in lib.si_last_error(), kw
    assert rotary(S=0) == 0  # nothing to do

    def pool(pages=8, H=2, P=4, D=64, prec=2, dtype=2, g=16, k=16, v=16, sk=16, sv=16):
        return (ctypes.c_int64 * 11)(pages, H, P, D, prec, dtype, g, k, v, sk, sv)

    bad = [dict(pages=0), dict(pages=1 << 40), dict(pages=1 << 30, P=4), dict(H=0), dict(H=65536), dict(P=0),
           dict(D=0), dict(D=513, g=1), dict(prec=4), dict(prec=-1), dict(dtype=3), dict(dtype=1 << 32),
           dict(g=24), dict(g=0), dict(k=0), dict(v=0), dict(sk=0), dict(sv=0), dict(k=8), dict(sv=24)]
    specs = [pool(**kw) for kw in bad] + [None]

    def write(spec=pool(), T=4, k=16, slots=16, turn=None, pos=16):
        return lib.si_pool_write(spec, k, 16, T, 128, 64, 128, 64, slots, turn, pos, 1, 1, None)

    def read(spec=pool(), T=4, slots=16, out=16, odt=0):
        return lib.si_pool_read(spec, slots, T, out, 16, odt, None)

    def attn(spec=pool(P=128), qdt=2, B=2, Hq=4, width=8, win=0, q=16, table=16, lens=16, out=16, ws=16,
             size=1 << 30):
        return lib.si_paged_attn(spec, q, qdt, B, Hq, 256, 64, table, 4, width, lens, win, 0.125, out, None, ws,
                                 size, None)

    for f, name in ((write, b"si_pool_write"), (read, b"si_pool_read"), (attn, b"si_paged_attn")):
        for spec in specs:
            assert f(spec=spec) == 1 and name in lib.si_last_error(), (name, spec and list(spec))
    for kw in (dict(T=-1), dict(T=1 << 31), dict(slots=None), dict(k=None), dict(turn=rotation(33)),
               dict(turn=rotation(0)), dict(turn=rotation(8, 0)), dict(turn=rotation(8), pos=None)):
        assert write(**kw) == 1 and b"si_pool_write" in lib.si_last_error(), kw
    assert write(T=0) == 0
    for kw in (dict(T=-1), dict(T=1 << 31), dict(slots=None), dict(out=None), dict(odt=4)):
        assert read(**kw) == 1 and b"si_pool_read" in lib.si_last_error(), kw
    assert read(T=0) == 0
    for kw in (dict(qdt=3), dict(Hq=3), dict(Hq=0), dict(B=-1), dict(B=1 << 30), dict(width=-1),
               dict(width=1 << 25), dict(win=-1), dict(win=1 << 31), dict(q=None), dict(table=None),
               dict(lens=None), dict(out=None), dict(ws=None), dict(ws=24), dict(size=8)):
        assert attn(**kw) == 1 and b"si_paged_attn" in lib.si_last_error(), kw
    assert attn(B=0) == 0
    size = lib.si_paged_attn_workspace_bytes
    assert size(1, 4, 2, 64, 4096, 0) > 0 and size(1, 4, 2, 64, 4096, 0) == size(9, 4, 2, 64, 1 << 20, 0)
    assert size(1, 4, 2, 64, 4096, 100) == 0 and size(1, 4, 2, 64, 100, 0) == 0
    assert size(1, 4, 3, 64, 4096, 0) == 0 and size(1, 4, 0, 64, 4096, 0) == 0


# ------------------------------------------------------------------- oracle
def test_oracle_rows_match_the_packed_oracle():
    """The pool's rows are the packed cache's: encode() against the C oracle."""
    g = torch.Generator().manual_seed(0)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        x = torch.randn(20, 48, generator=g).to(dtype)
        x[3] = 0
        q, s = R.encode(x, "int8", 16)
        oq, os_ = O.quant_rows_i8(to_np(x), DT[dtype])
        assert np.array_equal(q.numpy(), oq) and np.array_equal(to_np(s).ravel(), np.ravel(os_))
        q, s = R.encode(x, "int4", 16)
        oq, os_ = O.quant_rows_i4(to_np(x), DT[dtype], 16)
        assert np.array_equal(q.numpy(), O.pack_int4_rows(oq))
        assert np.array_equal(to_np(s).ravel(), np.ravel(os_))


def test_oracle_known_answers():
    q = torch.tensor([[[1.0, 0.0]], [[1.0, 0.0]], [[0.0, 1.0]]])
    k = torch.zeros(2, 1, 2, 2, dtype=torch.float64)
    v = torch.zeros_like(k)
    k[0, 0, 0] = torch.tensor([math.log(3.0), 0.0])
    v[0, 0, 0] = torch.tensor([4.0, 8.0])
    v[0, 0, 1] = torch.tensor([0.0, 4.0])
    k[1] = math.nan  # a page that only invalid entries could reach
    table = torch.tensor([[0, -1], [5, 0], [0, 0]], dtype=torch.int32)
    lengths = torch.tensor([4, 3, 0], dtype=torch.int32)
    out, lse, *_ = R.attend(q, k, v, table, lengths, 1.0)
    # positions 0, 1 of page 0 count, those of page -1 do not: weights 3/4, 1/4
    assert torch.allclose(out[0, 0], torch.tensor([3.0, 7.0], dtype=torch.float64))
    assert float(lse[0, 0]) == pytest.approx(math.log(4.0))
    # page 5 is outside, one position of page 0 is left
    assert torch.allclose(out[1, 0], torch.tensor([4.0, 8.0], dtype=torch.float64))
    # no position: zeros and -inf
    assert (out[2] == 0).all() and float(lse[2, 0]) == -math.inf
    out, *_ = R.attend(q[:1], k, v, table[:1], torch.tensor([2], dtype=torch.int32), 1.0, window=1)
    assert torch.allclose(out[0, 0], torch.tensor([0.0, 4.0], dtype=torch.float64))
    x = torch.tensor([[[1.0, 0.0, 5.0]]])
    turned = R.rotate(x, torch.tensor([1]), torch.tensor([math.pi / 2], dtype=torch.float64), gain=2.0)
    assert torch.allclose(turned, torch.tensor([[[0.0, 2.0, 5.0]]], dtype=torch.float64))
