"""Rows held in 4 bits (vdb_rows4_*, vectordb_amd.rows4) against a 64-bit restatement of the format."""
import ctypes as C

import numpy as np
import pytest

from vectordb_amd import _lib

torch = pytest.importorskip("torch")

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def values(codes, scales, dim):
    """[n, dim] float64 of codes [n, groups * 16] and scales [n, groups]."""
    nib = np.stack([codes & 15, codes >> 4], 2).reshape(codes.shape[0], -1)
    v = E2M1[nib & 7] * np.where(nib & 8, -1.0, 1.0)
    s = np.exp2(scales.astype(np.float64) - 127)
    s[scales == 255] = np.nan
    return (v * np.repeat(s, 32, 1))[:, :dim]


def packed(x):
    """The packing rule in 64 bits: (codes, scales) of rows x [n, dim]."""
    n, dim = x.shape
    g = -(-dim // 32)
    p = np.zeros((n, g * 32))
    p[:, :dim] = x
    p = p.reshape(n, g, 32)
    top = np.abs(p).max(2)
    bad = ~np.isfinite(top)
    f, e = np.frexp(np.where(bad, 0, top))
    e = np.where(f <= 0.75, e - 3, e - 2)
    byte = np.where(top == 0, 127, np.clip(127 + e, 1, 252))  # 6 * 2^125 is the largest such value in f32: saturates
    byte = np.where(bad, 255, byte)
    r = np.where(bad[:, :, None], 0, p) / np.exp2(np.where(bad, 0, byte - 127.0))[:, :, None]
    d = np.abs(np.abs(r)[..., None] - E2M1)
    near = d == d.min(-1, keepdims=True)
    # ties to the even code: of two neighbours the one whose lowest bit is 0
    code = np.where(near.sum(-1) > 1, np.argmax(near & (np.arange(8) % 2 == 0), -1), np.argmax(near, -1))
    code = code + np.where(np.signbit(r), 8, 0)
    code[bad] = 0
    code = code.reshape(n, -1).astype(np.uint8)
    return code[:, 0::2] | code[:, 1::2] << 4, byte.astype(np.uint8)


def random_rows(n, dim, seed, lo=118, hi=134):
    r = np.random.default_rng(seed)
    g = -(-dim // 32)
    codes = r.integers(0, 256, (n, g * 16), dtype=np.uint8)  # columns past dim hold anything
    return codes, r.integers(lo, hi, (n, g), dtype=np.uint8)


def products_bound(x, v):
    """A sum of len exact products in f32, in any order, each query in up to three exact parts: (3 len + 3) roundings of 2^-24."""
    return (3 * -(-v.shape[1] // 128) * 128 + 3) * 2.0 ** -24 * (np.abs(x) @ np.abs(v).T) + 1e-37


def test_refusals_without_a_device():
    l = _lib.lib()
    one = C.c_void_p(16)
    for args, word in [((one, one, 5, 0, one, 0, 1, 0, one), "dim"), ((one, one, 5, (1 << 20) + 1, one, 0, 1, 0, one), "dim"),
                       ((one, one, 1 << 31, 4, one, 0, 1, 4, one), "n must"), ((one, one, 5, 4, one, 3, 1, 4, one), "type"),
                       ((one, one, 5, 4, one, -1, 1, 4, one), "type"), ((one, one, 5, 4, one, 0, 65536, 4, one), "65535"),
                       ((None, one, 5, 4, one, 0, 1, 4, one), "codes"), ((C.c_void_p(8), one, 5, 4, one, 0, 1, 4, one), "codes"),
                       ((one, None, 5, 4, one, 0, 1, 4, one), "scales"), ((one, one, 5, 4, None, 0, 1, 4, one), "queries"),
                       ((one, one, 5, 4, C.c_void_p(18), 0, 1, 4, one), "queries"), ((one, one, 5, 4, one, 0, 1, 4, None), "out")]:
        assert l.vdb_rows4_products_device(*args, None) == _lib.VDB_ERR_INVALID
        assert word in l.vdb_last_error().decode()
    assert l.vdb_rows4_pack_device(None, 0, 3, 4, 4, one, one, None) == _lib.VDB_ERR_INVALID
    assert l.vdb_rows4_pack_device(one, 0, 3, 4, 4, C.c_void_p(4), one, None) == _lib.VDB_ERR_INVALID
    assert l.vdb_rows4_unpack_device(one, one, 3, 4, None, None) == _lib.VDB_ERR_INVALID
    # nothing to do is no error and touches no device
    assert l.vdb_rows4_products_device(None, None, 0, 4, None, 0, 1, 4, None, None) == _lib.VDB_OK
    assert l.vdb_rows4_products_device(None, None, 5, 4, None, 0, 0, 4, None, None) == _lib.VDB_OK
    assert l.vdb_rows4_pack_device(None, 0, 0, 4, 4, None, None, None) == _lib.VDB_OK


def test_python_refusals():
    from vectordb_amd.rows4 import Rows4

    with pytest.raises(ValueError):  # not on a device
        Rows4(torch.zeros((3, 16), dtype=torch.uint8), torch.zeros((3, 1), dtype=torch.uint8), 20)
    with pytest.raises(ValueError):
        Rows4.pack(torch.zeros((3, 20)))


def make(codes, scales, dim):
    from vectordb_amd.rows4 import Rows4

    return Rows4(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), dim)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,dim,nq", [(1, 1, 1), (15, 31, 2), (16, 32, 5), (17, 33, 6), (63, 100, 7), (65, 128, 8), (130, 129, 9),
                                      (257, 960, 1), (1000, 96, 16), (333, 1000, 17), (20, 4100, 3), (5000, 64, 33), (40, 2049, 40)])
def test_products(dtype, n, dim, nq):
    codes, scales = random_rows(n, dim, n + dim)
    rows = make(codes, scales, dim)
    x = torch.from_numpy(np.random.default_rng(nq).standard_normal((nq, dim)).astype(np.float32)).to(TYPES[dtype]).cuda()
    y = rows.products(x).cpu().numpy().astype(np.float64)
    v, xd = values(codes, scales, dim), x.cpu().double().numpy()
    assert y.shape == (nq, n)
    assert (np.abs(y - xd @ v.T) <= products_bound(xd, v)).all()
    one = rows.products(x[0])
    assert one.shape == (n,) and (np.abs(one.cpu().numpy() - xd[0] @ v.T) <= products_bound(xd[:1], v)[0]).all()


@pytest.mark.gpu
def test_products_f32_queries_keep_all_bits():
    """One row of a single 1: the product is the query's value itself, bit for bit, over the whole range of f32."""
    dim = 64
    codes = np.zeros((dim, 32), np.uint8)
    for i in range(dim):
        codes[i, i // 2] = 2 << 4 * (i % 2)  # value 1 at column i of row i
    rows = make(codes, np.full((dim, 2), 127, np.uint8), dim)
    bits = np.random.default_rng(3).integers(0, 1 << 32, (50, dim), dtype=np.uint32)
    bits = np.where((bits >> 23 & 0xFF) == 0xFF, np.uint32(0x3F800001), bits)
    bits = np.where((bits >> 23 & 0xFF) < 40, bits | np.uint32(0x10000000), bits)  # parts of smaller values would be subnormal
    bits[0, :4] = [0x7F7FFFFF, 0xFF7FFFFF, 0x3F7FFFFF, 0x80000000]
    x = bits.view(np.float32)
    y = rows.products(torch.from_numpy(x).cuda()).cpu().numpy()
    np.testing.assert_array_equal(y, x)


@pytest.mark.gpu
def test_products_strides_and_out():
    codes, scales = random_rows(70, 45, 1)
    rows = make(codes, scales, 45)
    wide = torch.randn(9, 101, device="cuda")
    v = values(codes, scales, 45)
    for x in (wide[:, 3:48], wide[::2, 1:46], torch.randn(45, 6, device="cuda").t(), torch.randn(45, device="cuda").expand(4, 45)):
        xd = x.cpu().double().numpy()
        out = torch.full((x.shape[0], 70), 7.0, device="cuda")
        assert rows.products(x, out=out) is out
        assert (np.abs(out.cpu().numpy() - xd @ v.T) <= products_bound(xd, v)).all()
    assert rows.products(wide[:0, :45]).shape == (0, 70)
    empty = make(np.zeros((0, 32), np.uint8), np.zeros((0, 2), np.uint8), 45)
    assert empty.products(wide[:, :45]).shape == (9, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_products_not_finite(dtype):
    codes, scales = random_rows(40, 70, 5)
    scales[7, 1] = 255
    rows = make(codes, scales, 70)
    x = torch.randn(4, 70).to(TYPES[dtype])
    x[1, 20], x[2, 69] = float("inf"), float("nan")
    y = rows.products(x.cuda()).cpu().numpy()
    v, xd = values(codes, scales, 70), x.double().numpy()
    with np.errstate(invalid="ignore"):
        ref = (xd[:, None, :] * v[None]).sum(2)
    np.testing.assert_array_equal(np.isnan(y), np.isnan(ref))
    np.testing.assert_array_equal(np.isinf(y), np.isinf(ref))
    np.testing.assert_array_equal(y[np.isinf(ref)], ref[np.isinf(ref)])
    assert np.isnan(y[:, 7]).all() and np.isnan(y[2]).all() and np.isfinite(np.delete(y[0], 7)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,dim", [(1, 1), (5, 32), (70, 100), (300, 960), (9, 4097)])
def test_pack_and_unpack(dtype, n, dim):
    from vectordb_amd.rows4 import Rows4

    r = np.random.default_rng(dim)
    x = (r.standard_normal((n, dim)) * np.exp2(r.integers(-10, 10, (n, 1)))).astype(np.float32)
    x[0, 0] = 0.0
    x = torch.from_numpy(x).to(TYPES[dtype])
    rows = Rows4.pack(x.cuda())
    codes, scales = packed(x.double().numpy())
    np.testing.assert_array_equal(rows.scales.cpu().numpy(), scales)
    got = values(rows.codes.cpu().numpy(), rows.scales.cpu().numpy(), dim)
    np.testing.assert_array_equal(got, values(codes, scales, dim))
    np.testing.assert_array_equal(rows.unpack().cpu().double().numpy(), got)
    # half a step at most: steps are 1/2 of the leading power of two (1/2 below 1), magnitudes reach 6 scales
    assert (np.abs(got - x.double().numpy()) <= np.repeat(np.exp2(scales - 127.0), 32, 1)[:, :dim]).all()


@pytest.mark.gpu
def test_pack_ties_edges_and_strides():
    from vectordb_amd.rows4 import Rows4

    x = np.zeros((6, 64), np.float32)
    x[0, :13] = [6, 5, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, 0.2500001, -5, -0.25, 4.9999995, 5.0000005]  # ties go to the even code
    x[1, 5], x[2, 40], x[3, :] = np.inf, np.nan, 0
    x[4, 0], x[4, 33] = 3.4e38, 1e-40
    x[5, :] = 1e-45
    wide = torch.zeros(6, 70).cuda()
    wide[:, 2:66] = torch.from_numpy(x)
    for src in (wide[:, 2:66], torch.from_numpy(x).t().contiguous().cuda().t()):
        rows = Rows4.pack(src)
        codes, scales = packed(x.astype(np.float64))
        np.testing.assert_array_equal(rows.scales.cpu().numpy(), scales)
        np.testing.assert_array_equal(rows.unpack().cpu().double().numpy(), values(codes, scales, 64))
    assert torch.isnan(rows.unpack()[1, :32]).all() and not torch.isnan(rows.unpack()[1, 32:]).any()


@pytest.mark.gpu
def test_beside_the_exact_scan():
    """As it would be used: the 4-bit rows pick candidates, whose exact distances (bruteforce.hpp:147-184) decide."""
    from vectordb_amd import datasets
    from vectordb_amd import index as vi
    from vectordb_amd.rows4 import Rows4

    x = datasets.clustered(4000, 96, 1)
    q = datasets.clustered(20, 96, 2)
    bf = vi.BruteforceSearch(vi.InnerProductSpace(96), 4000)
    bf.add_items(x)
    bf.to_device(0)
    xd, qd = torch.from_numpy(x).cuda(), torch.from_numpy(q).cuda()
    dist, label = bf.search_batch(qd, 10)
    rows = Rows4.pack(xd)
    score = rows.products(qd)
    v = rows.unpack().cpu().double().numpy()
    assert (np.abs(score.cpu().numpy() - q.astype(np.float64) @ v.T) <= products_bound(q.astype(np.float64), v)).all()
    # each product is off by at most |q| . |x - value|, so rows within twice the largest such error of the 10th best hold the answer
    off = (qd.abs().double() @ (xd.double() - rows.unpack().double()).abs().t()).max(1, keepdim=True).values.float()
    tenth = score.topk(10, 1).values[:, 9:]
    keep = score >= tenth - 2.001 * off
    assert keep.gather(1, label).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,dim,nq", [(8200 * 16 + 3, 96, 3), (8200 * 16 + 5, 300, 2), (8192 * 16, 129, 20), (600 * 16 + 1, 600, 5),
                                      (1500 * 16 + 7, 200, 18), (40, 30000, 2), (50, 9000, 16), (700, 2100, 32)])
def test_products_every_variant(dtype, n, dim, nq):
    """Sizes on both sides of every rule: many rows of one and of more blocks of columns, waves that share a tile, one and two
    tiles of queries, queries too large for LDS."""
    codes, scales = random_rows(n, dim, n % 1000 + dim)
    rows = make(codes, scales, dim)
    x = torch.from_numpy(np.random.default_rng(nq).standard_normal((nq, dim)).astype(np.float32)).to(TYPES[dtype])
    y = rows.products(x.cuda())
    rowsd = torch.from_numpy(values(codes, scales, dim))
    ref, size = x.double() @ rowsd.t(), x.double().abs() @ rowsd.abs().t()
    tol = (3 * -(-dim // 128) * 128 + 3) * 2.0 ** -24 * size + 1e-37
    assert ((y.cpu().double() - ref).abs() <= tol).all()
    again = rows.products(x.cuda())
    assert torch.equal(y, again)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,dim", [(40, 70), (40, 31), (5, 1), (40, 97), (140_000, 100), (9000, 700), (300, 2049)])
@pytest.mark.parametrize("byte", [0, 1, 252, 253, 254])
def test_products_scales_at_the_ends(dtype, n, dim, byte):
    """The smallest and largest scales, with codes past the last column that are infinite under them: those are never used."""
    r = np.random.default_rng(byte + dim)
    g = -(-dim // 32)
    codes = r.integers(0, 256, (n, g * 16), dtype=np.uint8)
    scales = r.integers(118, 134, (n, g), dtype=np.uint8)
    scales[::3, -1] = byte
    if byte >= 253:  # in the columns that are used, 0 and 0.5 only: finite
        for c in range(dim - (g - 1) * 32):
            codes[:, (g - 1) * 16 + c // 2] &= 0x9F if c % 2 else 0xF9
    rows = make(codes, scales, dim)
    x = torch.from_numpy((r.standard_normal((3, dim)) * 2.0 ** -6).astype(np.float32)).to(TYPES[dtype])
    y = rows.products(x.cuda()).cpu().numpy().astype(np.float64)
    v, xd = values(codes, scales, dim), x.double().numpy()
    assert (np.abs(y - xd @ v.T) <= products_bound(xd, v)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n,dim,nq", [(40, 64, 5), (600, 960, 2), (140_000, 100, 3)])
def test_products_of_the_smallest_queries(n, dim, nq):
    """f32 queries near and below the least normal number: what lies below 2^-133 in a value may be cut off, and nothing else."""
    codes, scales = random_rows(n, dim, n + dim, lo=127, hi=150)
    rows = make(codes, scales, dim)
    r = np.random.default_rng(nq)
    x = (r.standard_normal((nq, dim)) * np.exp2(r.integers(-149, -100, (nq, dim)))).astype(np.float32)
    x[0, :8] = [2.0 ** -149, -2.0 ** -133, 2.0 ** -126, 2.0 ** -133 * 1.5, 0.0, 2.0 ** -110 * (1 + 2.0 ** -23), 2.0 ** -127, -2.0 ** -148]
    y = rows.products(torch.from_numpy(x).cuda()).cpu().numpy().astype(np.float64)
    v, xd = values(codes, scales, dim), x.astype(np.float64)
    size = np.abs(xd) @ np.abs(v).T
    # (products_bound's own 1e-37 is left out: a step of the smallest results is 2^-149, one for each of the roundings)
    steps = 3 * -(-dim // 128) * 128 + 3
    assert (np.abs(y - xd @ v.T) <= steps * (2.0 ** -24 * size + 2.0 ** -149) + 2.0 ** -133 * np.abs(v).sum(1)).all()
