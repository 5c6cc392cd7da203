"""The 8-bit key / value memory (vdb_kv_*, vectordb_amd.memory) against restatements on the CPU: the append bit for bit
(every step of it is a single rounding), the attention in 64 bits."""
import ctypes as C
import math

import numpy as np
import pytest

from vectordb_amd import _lib

torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn
EPS = 2.0 ** -24


# ---- restatements ---------------------------------------------------------------------------------

def turn(x, cos, sin, interleaved):
    """x [..., dim] f32 CPU, cos / sin [half] f32: the pair (a, b) -> (a c - b s, b c + a s), each operation rounded."""
    half = cos.shape[0]
    out = x.clone()
    ia, ib = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., ia], x[..., ib]
    out[..., ia] = a * cos - b * sin
    out[..., ib] = b * cos + a * sin
    return out


def fit(top):
    """The smallest power of two s with top <= 448 s, at least 2^-100."""
    if top == 0:
        return 2.0 ** -100
    e = math.ceil(math.log2(top / 448)) - 2
    while top > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** max(e, -100)


def to_code(x):
    """f32 -> e4m3, infinities like NaN."""
    return torch.where(torch.isfinite(x), x, torch.nan).to(E4M3)


def append_ref(k, scale, x, table, lengths, offsets, page, cos=None, sin=None, interleaved=False):
    """One side (keys, or values without cos) of the append on CPU tensors, in place.  x [T, H, D]."""
    pages, heads = scale.shape
    x = x.float()
    for b, n_held in enumerate(lengths):
        lo, hi = offsets[b], offsets[b + 1]
        if hi <= lo or lo < 0 or hi > x.shape[0]:
            continue
        start = n_held - (hi - lo)
        for p in range(max(start, 0) // page, table.shape[1]):
            at = [t for t in range(max(start, 0, p * page), min(n_held, (p + 1) * page)) if cos is None or t < cos.shape[0]]
            pid = int(table[b, p])
            if not at or pid < 0 or pid >= pages:
                continue
            rows = torch.stack([x[lo + t - start] if cos is None else turn(x[lo + t - start], cos[t], sin[t], interleaved) for t in at])  # [n, H, D]
            r0 = max(start, 0) - p * page if p == max(start, 0) // page else 0
            for h in range(heads):
                mag = rows[:, h].abs()
                mag = mag[torch.isfinite(mag)]
                s = fit(float(mag.max()) if mag.numel() else 0.0)
                old = float(scale[pid, h])
                if r0 and old > s:
                    s = old
                if r0 and s != old:
                    k[pid, h, :r0] = (k[pid, h, :r0].float() * np.float32(old / s)).to(E4M3)
                scale[pid, h] = s
                k[pid, h, r0:r0 + len(at)] = to_code(rows[:, h] / np.float32(s))


def attend_ref(q, k, v, ks, vs, table, lengths, offsets, page, scale, window=0, select=None):
    """-> out [T, Hq, D] f64, lse [T, Hq], and the bounds sum p |v| and sum |q| |k| scale that tolerances need."""
    T, hq, D = q.shape
    pages, H = ks.shape
    G = hq // H
    out, lse = torch.zeros(T, hq, D, dtype=torch.float64), torch.full((T, hq), -math.inf, dtype=torch.float64)
    mass, size, count = torch.zeros(T, hq, D, dtype=torch.float64), torch.zeros(T, hq, dtype=torch.float64), 1
    for b, n_held in enumerate(lengths):
        lo, hi = offsets[b], offsets[b + 1]
        if hi <= lo or lo < 0 or hi > T or n_held == 0:
            continue
        pos = torch.arange(n_held - (hi - lo), n_held)
        for h in range(H):
            at = select[b, h] if select is not None else torch.arange(n_held)
            at = at[(at >= 0) & (at < min(n_held, page * table.shape[1]))]
            pid = table[b].long()[at // page]
            at, pid = at[(pid >= 0) & (pid < pages)], pid[(pid >= 0) & (pid < pages)]
            if not len(at):
                continue
            hidden = torch.zeros(hi - lo, len(at), dtype=torch.bool)
            if select is None:
                hidden |= at[None, :] > pos[:, None]
                if window:
                    hidden |= at[None, :] <= pos[:, None] - window
            kk = k.view(torch.uint8)[pid, h, at % page].view(E4M3).double() * ks[pid, h].double()[:, None]
            vv = v.view(torch.uint8)[pid, h, at % page].view(E4M3).double() * vs[pid, h].double()[:, None]
            qq = q[lo:hi, h * G:(h + 1) * G].double()
            s = (qq @ kk.t() * scale).masked_fill(hidden[:, None, :], -math.inf)  # [new, G, tokens]
            p = torch.softmax(s, 2).masked_fill((hidden.all(1))[:, None, None], 0.0)
            lost = ~hidden[:, None, :, None] & torch.isnan(vv)[None, None]  # a NaN that is seen; one that is not has no effect
            o = p @ vv.nan_to_num() if not torch.isnan(vv).any() else torch.where(lost.any(2), torch.nan, p @ vv.nan_to_num())
            out[lo:hi, h * G:(h + 1) * G] = o
            mass[lo:hi, h * G:(h + 1) * G] = p @ vv.nan_to_num().abs()
            lse[lo:hi, h * G:(h + 1) * G] = torch.logsumexp(s, 2)
            size[lo:hi, h * G:(h + 1) * G] = (qq.abs() @ kk.abs().t() * abs(scale)).masked_fill(hidden[:, None, :], 0.0).amax(2)
            count = max(count, int((~hidden).sum(1).max()))
    return out, lse, mass, size, count


def check_attend(got, lse, ref, dtype):
    """A score is a sum of D exact products in f32 (D + 8 roundings of 2^-24 of the magnitudes it adds, three parts of an f32 query
    included), p and the softmax's sum follow it; p is rounded to bf16 (results in bf16: half a step, 2^-8) or to parts of it (f16:
    2^-15, f32: 2^-22); sums over n tokens go through lanes, steps of 128 and waves (n / 32 + 64 roundings); the result is rounded."""
    out, ref_lse, mass, size, n = ref
    D = got.shape[-1]
    score = (3 * D + 16) * EPS * size
    part = {torch.float32: 2.0 ** -22, torch.float16: 2.0 ** -15, torch.bfloat16: 2.0 ** -8}[dtype]
    many = (n / 32 + 64) * EPS
    tol = (2 * score[..., None] + part + 2 * many) * mass * 1.01 + torch.finfo(dtype).eps / 2 * 1.01 * out.abs() + (6e-8 if dtype == torch.float16 else 1e-38)
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(out))
    bad = (got - out).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} values off, worst {((got - out).abs() / tol).nan_to_num().max():.2f} times the tolerance"
    if lse is not None:
        lse = lse.double().cpu()
        seen = torch.isfinite(ref_lse)
        assert torch.equal(lse[~seen].nan_to_num(nan=7.0), ref_lse[~seen].nan_to_num(nan=7.0))
        assert ((lse - ref_lse).abs()[seen] <= (score + many + 4 * EPS * (ref_lse.abs() + size))[seen]).all()


# ---- inputs ------------------------------------------------------------------------------------------

def random_codes(shape, g):
    return (torch.randn(shape, generator=g) * 90).clamp(-448, 448).to(E4M3)


class Setup:
    """A memory on the CPU: random pages, shuffled tables."""

    def __init__(self, lengths, page, heads, dim, seed=0, spare=3, width=None):
        g = torch.Generator().manual_seed(seed)
        self.g, self.page, self.heads, self.dim = g, page, heads, dim
        need = [-(-n // page) for n in lengths]
        width = max(max(need), 1) if width is None else width
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=g).int()
        self.table = torch.full((len(lengths), width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :min(n, width)] = order[at:at + min(n, width)]
            at += n
        self.lengths = list(lengths)
        self.k, self.v = random_codes((pages, heads, page, dim), g), random_codes((pages, heads, page, dim), g)
        self.ks = torch.exp2(torch.randint(-8, -4, (pages, heads), generator=g).float())
        self.vs = torch.exp2(torch.randint(-8, -4, (pages, heads), generator=g).float())

    def memory(self):
        from vectordb_amd.memory import KeyValueMemory

        return KeyValueMemory.from_tensors(self.k.cuda(), self.v.cuda(), self.ks.cuda(), self.vs.cuda())

    def on_gpu(self):
        return self.table.cuda(), torch.tensor(self.lengths, dtype=torch.int32, device="cuda")

    def randn(self, *shape, dtype=torch.float32):
        return torch.randn(shape, generator=self.g).to(dtype)


def offsets_of(new):
    return [sum(new[:i]) for i in range(len(new) + 1)]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def angles(n, half):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))
    return a.cos().float(), a.sin().float()


def same_codes(a, b):
    a, b = a.cpu().float(), b.float()
    return torch.equal(a.nan_to_num(nan=1e9), b.nan_to_num(nan=1e9))


# ---- refusals (no device) ------------------------------------------------------------------------------

def good():
    m = _lib.KvMemoryStruct(16, 16, 16, 16, 10, 2, 16, 64)
    b = _lib.KvBatchStruct(16, 16, None, 3, 4, 3, 1)
    return m, b


def test_attend_refusals_without_a_device():
    l = _lib.lib()

    def call(m, b, dtype=0, q=16, ts=128, hs=64, qh=4, window=0, select=None, n=0, out=16, work=16, size=1 << 40):
        return l.vdb_kv_attend_device(m, b, dtype, q, ts, hs, qh, 1.0, window, select, n, out, None, work, size, None)

    cases = []
    for field, value, word in [("page_tokens", 8, "page_tokens"), ("page_tokens", 24, "page_tokens"), ("page_tokens", 2048, "page_tokens"),
                               ("dim", 48, "dim"), ("dim", 0, "dim"), ("dim", 288, "dim"), ("heads", 0, "heads"), ("heads", 40000, "heads"),
                               ("pages", 1 << 31, "pages"), ("k", None, "k"), ("v", 8, "v"), ("k_scale", None, "k_scale"), ("v_scale", 2, "v_scale")]:
        m, b = good()
        setattr(m, field, value)
        cases.append((call(m, b), word))
    for field, value, word in [("count", 65536, "65535"), ("table_width", 0, "table_width"), ("tokens", 1 << 31, "tokens"), ("tokens", 4, "offsets"),
                               ("table", None, "table"), ("lengths", None, "lengths"), ("offsets", 2, "offsets")]:
        m, b = good()
        setattr(b, field, value)
        cases.append((l.vdb_kv_attend_device(m, b, 0, 16, 128, 64, 4, 1.0, 0, None, 0, 16, None, 16, 1 << 40, None), word))
    m, b = good()
    b.table_width = 1000  # so many tokens that a workspace is needed
    for kw, word in [(dict(dtype=3), "type"), (dict(q=None), "queries"), (dict(q=8), "queries"), (dict(ts=4), "strides"), (dict(hs=65), "strides"),
                     (dict(qh=3), "q_heads"), (dict(qh=0), "q_heads"), (dict(window=1 << 31), "window"), (dict(out=None), "out"), (dict(out=8), "out"),
                     (dict(select=16, n=4, window=3), "window"), (dict(select=4, n=4), "select"), (dict(select=16, n=1 << 31), "n_select"), (dict(select=16, n=0), "n_select"),
                     (dict(size=0), "workspace"), (dict(work=None), "workspace")]:
        cases.append((call(m, b, **kw), word))
        assert word in l.vdb_last_error().decode(), kw
    assert all(rc == _lib.VDB_ERR_INVALID for rc, _ in cases), cases
    assert l.vdb_kv_attend_device(None, b, 0, 16, 128, 64, 4, 1.0, 0, None, 0, 16, None, 16, 0, None) == _lib.VDB_ERR_INVALID
    assert l.vdb_kv_attend_device(m, None, 0, 16, 128, 64, 4, 1.0, 0, None, 0, 16, None, 16, 0, None) == _lib.VDB_ERR_INVALID
    b.offsets = 16
    assert call(m, b, select=16, n=4) == _lib.VDB_ERR_INVALID
    b.offsets, b.count, b.tokens = None, 0, 0
    assert call(m, b, q=None, out=None) == _lib.VDB_OK  # no sequences: nothing to do


def test_append_refusals_without_a_device():
    l = _lib.lib()

    def call(dtype=0, k=16, kt=128, kh=64, v=16, vt=128, vh=64, cos=16, sin=16, pos=9, rot=32, q=16, qt=128, qh=64, heads=4, out=16, change=()):
        m, b = good()
        for o, f, x in change:
            setattr(m if o == "m" else b, f, x)
        return l.vdb_kv_append_device(m, b, dtype, k, kt, kh, v, vt, vh, cos, sin, pos, rot, 0, q, qt, qh, heads, out, None)

    for kw, word in [(dict(dtype=7), "type"), (dict(rot=8), "rot_dims"), (dict(rot=80), "rot_dims"), (dict(rot=0), "rot_dims"), (dict(k=None), "keys"),
                     (dict(k=24), "keys"), (dict(kt=4), "keys"), (dict(kh=1), "keys"), (dict(v=None), "values"), (dict(vt=12), "values"),
                     (dict(cos=None), "cos"), (dict(sin=8), "sin"), (dict(q=8), "queries"), (dict(qt=9), "queries"), (dict(heads=0), "q_heads"),
                     (dict(out=None), "q_out"), (dict(change=[("m", "dim", 40)]), "dim"), (dict(change=[("b", "count", 70000)]), "65535"),
                     (dict(change=[("b", "tokens", 5)]), "offsets"), (dict(change=[("b", "table", None)]), "table")]:
        assert call(**kw) == _lib.VDB_ERR_INVALID, kw
        assert word in l.vdb_last_error().decode(), kw
    assert call(change=[("b", "count", 0), ("b", "tokens", 0)], k=None, v=None) == _lib.VDB_OK


def test_python_refusals_without_a_device():
    from vectordb_amd.memory import KeyValueMemory

    k = torch.zeros(4, 2, 16, 64, dtype=torch.uint8).view(E4M3)
    s = torch.ones(4, 2)
    for args in [(k, k, s, s), (k, k[:3], s, s), (k.float(), k.float(), s, s), (k, k, s[:, :1], s)]:
        with pytest.raises(ValueError):
            KeyValueMemory.from_tensors(*args)


@pytest.mark.gpu
def test_python_refusals():
    from vectordb_amd.memory import KeyValueMemory

    mem = KeyValueMemory(6, 16, 2, 64)
    table, lengths = ints([[0, 1], [2, 3]]), ints([5, 20])
    q = torch.zeros(2, 4, 64, device="cuda")
    kv = torch.zeros(2, 2, 64, device="cuda")
    for call in [lambda: mem.attend(q[:, :3], table, lengths), lambda: mem.attend(q[:, :, :32], table, lengths), lambda: mem.attend(q.double(), table, lengths),
                 lambda: mem.attend(q.cpu(), table, lengths), lambda: mem.attend(q, table.long(), lengths), lambda: mem.attend(q, table[:1], lengths),
                 lambda: mem.attend(q[:1], table, lengths), lambda: mem.attend(q, table, lengths.cpu()), lambda: mem.attend(q, table, lengths, window=-1),
                 lambda: mem.attend(q, table, lengths, offsets=ints([0, 2])), lambda: mem.attend(q, table, lengths, select=torch.zeros(2, 2, 3, device="cuda")),
                 lambda: mem.attend(q, table, lengths, window=3, select=torch.zeros(2, 2, 3, dtype=torch.int64, device="cuda")),
                 lambda: mem.attend(q, table, lengths, offsets=ints([0, 1, 2]), select=torch.zeros(2, 2, 3, dtype=torch.int64, device="cuda")),
                 lambda: mem.attend(q[:, :0], table, lengths), lambda: mem.append(kv, kv[:1], table, lengths), lambda: mem.append(kv, kv.half(), table, lengths),
                 lambda: mem.append(kv[:, :1], kv[:, :1], table, lengths), lambda: mem.append(kv, kv, table, lengths, cos=torch.zeros(9, 16, device="cuda")),
                 lambda: mem.append(kv, kv, table, lengths, queries=q.half()), lambda: mem.append(kv, kv, table, lengths, queries=q[:1]),
                 lambda: KeyValueMemory(6, 24, 2, 64), lambda: KeyValueMemory(6, 16, 2, 40)]:
        with pytest.raises(ValueError):
            call()
    c = torch.zeros(9, 20, device="cuda")
    with pytest.raises(_lib.VdbError):  # 40 turned dimensions
        mem.append(kv, kv, table, lengths, cos=c, sin=c)


# ---- append ------------------------------------------------------------------------------------------------

APPENDS = [
    # lengths after, new tokens, page, heads, q heads, dim, turned, interleaved
    ([1], [1], 16, 1, 1, 32, 0, False),
    ([17, 16, 1, 40], [1, 1, 1, 1], 16, 2, 4, 64, 64, False),
    ([70, 33, 5, 128], [70, 20, 0, 64], 32, 3, 3, 96, 48, False),
    ([100, 64, 65], [37, 64, 1], 64, 2, 10, 128, 128, True),
    ([31, 200], [31, 150], 128, 1, 8, 160, 32, True),
    ([90], [61], 16, 4, 4, 256, 256, False),
    ([10, 0, 40], [15, 0, 3], 16, 2, 2, 192, 16, False),  # five tokens at negative positions: dropped
    ([1500], [1100], 1024, 1, 2, 32, 32, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: "-".join(map(str, c[2:7])) + "-" + str(len(c[0])))
def test_append(dtype, case):
    held, new, page, heads, hq, dim, rot, inter = case
    t = TYPES[dtype]
    s = Setup(held, page, heads, dim, seed=dim + page)
    off = offsets_of(new)
    total = off[-1] + 2  # two rows of no sequence
    k, v, q = s.randn(total, heads, dim, dtype=t) * 3, s.randn(total, heads, dim, dtype=t) * 40, s.randn(total, hq, dim, dtype=t)
    cos, sin = angles(max(held), rot // 2) if rot else (None, None)
    single = all(n == 1 for n in new)
    if single:
        k, v, q, total = k[:-2], v[:-2], q[:-2], total - 2
    mem = s.memory()
    table, lengths = s.on_gpu()
    got = mem.append(k.cuda(), v.cuda(), table, lengths, offsets=None if single else ints(off), max_new=max(new), queries=q.cuda(),
                     cos=None if cos is None else cos.cuda(), sin=None if sin is None else sin.cuda(), interleaved=inter)
    append_ref(s.k, s.ks, k, s.table, held, off, page, cos, sin, inter)
    append_ref(s.v, s.vs, v, s.table, held, off, page)
    assert torch.equal(mem.k_scale.cpu(), s.ks) and torch.equal(mem.v_scale.cpu(), s.vs)
    assert same_codes(mem.k, s.k) and same_codes(mem.v, s.v)  # the pages of nobody and the rows behind the last token included
    want = q.clone()
    for b, n in enumerate(new):
        for i in range(n):
            pos = held[b] - n + i
            if rot:
                want[off[b] + i] = turn(q[off[b] + i].float(), cos[pos], sin[pos], inter).to(t) if pos >= 0 else torch.full_like(q[0], float("nan"))
    assert same_codes(got, want.float())


@pytest.mark.gpu
def test_append_token_by_token():
    """Growing magnitudes raise a page's scale again and again; each time the older rows are rounded to it once more."""
    page, heads, dim = 16, 2, 64
    s = Setup([40], page, heads, dim, seed=5)
    mem = s.memory()
    table = s.table.cuda()
    for n in range(1, 41):
        k = s.randn(1, heads, dim) * 1.3 ** n * 1e-3
        v = s.randn(1, heads, dim) * 0.8 ** n
        mem.append(k.cuda(), v.cuda(), table, ints([n]))
        append_ref(s.k, s.ks, k, s.table, [n], [0, 1], page)
        append_ref(s.v, s.vs, v, s.table, [n], [0, 1], page)
    assert same_codes(mem.k, s.k) and same_codes(mem.v, s.v) and torch.equal(mem.k_scale.cpu(), s.ks)


@pytest.mark.gpu
def test_append_values_at_the_edges():
    page, heads, dim = 16, 1, 32
    s = Setup([20, 30, 16, 16, 3, 16], page, heads, dim, seed=6)
    new = [20, 3, 16, 16, 3, 16]
    k = s.randn(sum(new), heads, dim)
    off = offsets_of(new)
    k[0, 0, 3], k[1, 0, 4], k[2, 0, 5] = float("inf"), float("-inf"), float("nan")
    k[off[2]:off[3]] = 0.0
    k[off[3]:off[4]] *= 1e37
    k[off[3], 0, 0] = torch.finfo(torch.float32).max
    k[off[4]:off[5]] = float("nan")
    k[off[5]:] *= 1e-38
    k[off[1], 0, 0] = 448.0 * 2 ** -3  # the largest code exactly
    mem = s.memory()
    table, lengths = s.on_gpu()
    mem.append(k.cuda(), -k.cuda(), table, lengths, offsets=ints(off), max_new=20)
    append_ref(s.k, s.ks, k, s.table, s.lengths, off, page)
    append_ref(s.v, s.vs, -k, s.table, s.lengths, off, page)
    assert torch.equal(mem.k_scale.cpu(), s.ks) and torch.isfinite(mem.k_scale).all()
    assert same_codes(mem.k, s.k) and same_codes(mem.v, s.v)


@pytest.mark.gpu
def test_append_bad_tables_and_strides():
    """Absent pages, tables that are too short, positions beyond the angles, offsets out of range, a wrong max_new, views."""
    page, heads, dim, hq = 16, 2, 64, 4
    s = Setup([100, 50, 60, 20], page, heads, dim, seed=7, width=5)
    s.table[0, 2], s.table[1, 0], s.table[2, 1] = -7, 1000000, s.ks.shape[0]
    new = [90, 50, 30, 20]
    off = offsets_of(new)
    fused = s.randn(off[-1] + 3, hq + 2 * heads, dim, dtype=torch.bfloat16)
    q, k, v = fused[:, :hq], fused[:, hq:hq + heads], fused[:, hq + heads:]
    cos, sin = angles(66, 32)
    bad = off[:-1] + [off[-1] + 10]  # the last sequence claims rows that are not there
    mem = s.memory()
    f = fused.cuda()
    table, lengths = s.on_gpu()
    got = mem.append(f[:, hq:hq + heads], f[:, hq + heads:], table, lengths, offsets=ints(bad), max_new=1, queries=f[:, :hq], cos=cos.cuda(), sin=sin.cuda())
    append_ref(s.k, s.ks, k, s.table, s.lengths, bad, page, cos, sin)
    append_ref(s.v, s.vs, v, s.table, s.lengths, bad, page)
    assert same_codes(mem.k, s.k) and same_codes(mem.v, s.v) and torch.equal(mem.k_scale.cpu(), s.ks) and torch.equal(mem.v_scale.cpu(), s.vs)
    got = got.cpu()
    assert torch.isnan(got[off[0] + 66 - 10:off[1]].float()).all() and torch.equal(got[off[3]:], q[off[3]:])
    assert torch.equal(got[off[2]:off[3]], torch.stack([turn(q[off[2] + i].float(), cos[30 + i], sin[30 + i], False).bfloat16() for i in range(30)]))
    # a head stride that is no multiple of 8, a negative step, an odd start: copied on the way
    odd = torch.randn(4, heads, dim + 1, device="cuda")
    for x in (odd[:, :, :dim], odd[:, :, 1:], odd[:, :, :dim].transpose(0, 1).contiguous().transpose(0, 1)):
        a, b = Setup([5, 6, 7, 8], page, heads, dim, seed=8), Setup([5, 6, 7, 8], page, heads, dim, seed=8)
        mem = a.memory()
        table, lengths = a.on_gpu()
        mem.append(x, x, table, lengths)
        append_ref(b.k, b.ks, x.cpu(), b.table, b.lengths, [0, 1, 2, 3, 4], page)
        assert same_codes(mem.k, b.k)


# ---- attend -----------------------------------------------------------------------------------------------

ATTENDS = [
    # lengths, new tokens, page, heads, q heads, dim, window
    ([1], [1], 16, 1, 1, 32, 0),
    ([16, 1, 33, 0], [1, 1, 1, 1], 16, 2, 2, 64, 0),
    ([257, 31, 129], [1, 1, 1], 32, 3, 12, 96, 0),
    ([500, 90], [1, 1], 64, 2, 32, 128, 0),          # 16 query heads a key head
    ([300], [1], 16, 1, 20, 160, 0),                 # 20: more than one tile of rows
    ([700, 64, 65], [1, 1, 1], 128, 2, 8, 256, 0),
    ([1000, 3], [1, 1], 64, 2, 4, 128, 100),
    ([60, 130], [60, 33], 16, 2, 4, 64, 0),          # chunks
    ([200, 7, 40], [90, 7, 0], 32, 1, 3, 128, 0),
    ([150], [150], 64, 2, 2, 192, 17),
    ([70], [40], 16, 1, 5, 224, 1),                  # a window of one token: the value itself
    ([10], [20], 16, 1, 2, 32, 0),                   # ten queries at negative positions see nothing
    ([5000], [3], 64, 1, 4, 128, 0),
    ([2000], [1], 1024, 1, 1, 64, 0),
    ([300, 290], [129, 128], 16, 2, 8, 128, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("case", ATTENDS, ids=lambda c: f"{c[0][0]}-{c[1][0]}-p{c[2]}-h{c[3]}-{c[4]}-d{c[5]}-w{c[6]}")
def test_attend(dtype, case):
    held, new, page, heads, hq, dim, window = case
    t = TYPES[dtype]
    s = Setup(held, page, heads, dim, seed=dim + page + len(held))
    off = offsets_of(new)
    single = all(n == 1 for n in new)
    total = off[-1] + (0 if single else 2)
    q = s.randn(total, hq, dim, dtype=t)
    mem = s.memory()
    table, lengths = s.on_gpu()
    scale = dim ** -0.5
    out, lse = mem.attend(q.cuda(), table, lengths, offsets=None if single else ints(off), max_new=max(new), window=window, return_lse=True)
    assert out.dtype == t and out.shape == q.shape
    ref = attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, off, page, scale, window)
    check_attend(out[:off[-1]], lse[:off[-1]], [x[:off[-1]] if torch.is_tensor(x) else x for x in ref], t)
    assert not out[off[-1]:].any()
    # offsets given and not given, lse asked for or not: the same bits
    again = mem.attend(q[:off[-1]].cuda(), table, lengths, offsets=ints(off), max_new=max(new), window=window)
    if single:
        check_attend(again, None, ref, t)
    else:
        assert torch.equal(again, out[:off[-1]])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("heads,hq,dim,page,n", [(1, 1, 32, 16, 1), (2, 8, 128, 64, 100), (3, 3, 96, 16, 33), (2, 40, 64, 32, 300)])
def test_attend_selected(dtype, heads, hq, dim, page, n):
    held = [400, 1, 77, 0]
    s = Setup(held, page, heads, dim, seed=n)
    t = TYPES[dtype]
    q = s.randn(4, hq, dim, dtype=t)
    select = torch.randint(0, 400, (4, heads, n), generator=s.g)
    select[:, :, n // 2:n // 2 + 2] = -1                      # a search's padding
    select[0, :, -1] = 2 ** 40
    if n > 10:
        select[0, :, 3] = select[0, :, 4] = 7                 # the same token twice counts twice
        select[2, 0] = -1                                     # nothing at all
    mem = s.memory()
    table, lengths = s.on_gpu()
    out, lse = mem.attend(q.cuda(), table, lengths, select=select.cuda(), return_lse=True)
    check_attend(out, lse, attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, [0, 1, 2, 3, 4], page, dim ** -0.5, 0, select), t)
    none = mem.attend(q.cuda(), table, lengths, select=select.cuda()[:, :, :0])
    assert not none.any()


@pytest.mark.gpu
@pytest.mark.parametrize("new,window", [([1, 1], 0), ([1, 1], 20), ([30, 40], 0), ([64, 100], 25), ([100, 10], 0)])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_attend_what_is_not_seen_has_no_effect(dim, new, window):
    """NaN codes, scales and queries where the mask leaves them out: the rows behind the last token, the future, before the
    window, the pages of nobody; and a NaN that IS seen reaches every query that sees it, and no other."""
    held, page, heads, hq = [130, 190], 16, 2, 6
    s = Setup(held, page, heads, dim, seed=11)
    off = offsets_of(new)
    k8, v8 = s.k.view(torch.uint8), s.v.view(torch.uint8)
    used = torch.zeros(s.ks.shape[0], page, dtype=torch.bool)
    for b, n in enumerate(held):
        for tok in range(n):
            used[s.table[b, tok // page].long(), tok % page] = True
    for c in (k8, v8):
        c.copy_(torch.where(used[:, None, :, None], c, torch.tensor(0x7F, dtype=torch.uint8)))
    s.ks[~used.any(1)] = float("nan")
    s.vs[~used.any(1)] = float("inf")
    # tokens that only the later queries of a chunk see, or that the window has left behind for them
    for b, tok, d in [(0, 129, 3), (0, 110, 0), (1, 170, dim - 1), (1, 150, 7), (1, 189, 20), (0, 60, 1)]:
        v8[s.table[b, tok // page].long(), 0, tok % page, d] = 0xFF
    k8[s.table[0, 120 // page].long(), 1, 120 % page, 5] = 0x7F
    q = s.randn(off[-1], hq, dim, dtype=torch.bfloat16)
    q[off[-1] - 1, 4, 9] = float("nan")
    mem = s.memory()
    table, lengths = s.on_gpu()
    out, lse = mem.attend(q.cuda(), table, lengths, offsets=None if max(new) == 1 else ints(off), max_new=max(new), window=window, return_lse=True)
    ref = attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, off, page, dim ** -0.5, window)
    check_attend(out, lse, ref, torch.bfloat16)


@pytest.mark.gpu
def test_attend_absent_pages_short_tables_and_views():
    held, page, heads, hq, dim = [100, 90, 200], 16, 2, 4, 64
    s = Setup(held, page, heads, dim, seed=12, width=8)
    s.table[0, 0], s.table[0, 3], s.table[1, 5] = -1, 2 ** 31 - 1, s.ks.shape[0]
    fused = s.randn(3, hq + 4, dim + 8, dtype=torch.float16)
    q = fused[:, 2:2 + hq, 8:]
    mem = s.memory()
    table, lengths = s.on_gpu()
    f = fused.cuda()
    out, lse = mem.attend(f[:, 2:2 + hq, 8:], table, lengths, return_lse=True)
    check_attend(out, lse, attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, [0, 1, 2, 3], page, dim ** -0.5), torch.float16)
    off = [0, 2, 2, 9]  # the last one claims rows that are not there: none
    out = mem.attend(f[:, 2:2 + hq, 8:], table, lengths, offsets=ints(off), max_new=1)
    ref = attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, off, page, dim ** -0.5)
    check_attend(out, None, ref, torch.float16)
    s.table[:] = -1
    out, lse = mem.attend(f[:, 2:2 + hq, 8:], s.table.cuda(), lengths, return_lse=True)
    assert not out.any() and (lse == -math.inf).all()


@pytest.mark.gpu
def test_attend_far_scores():
    """Scores of hundreds: the running maximum has to carry them; and equal scores: the mean of the values."""
    held, page, heads, dim = [333], 16, 1, 64
    s = Setup(held, page, heads, dim, seed=13)
    mem = s.memory()
    table, lengths = s.on_gpu()
    for mul in (100.0, 0.0, -100.0):
        q = s.randn(1, 2, dim) * mul
        out, lse = mem.attend(q.cuda(), table, lengths, return_lse=True)
        check_attend(out, lse, attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, [0, 1], page, dim ** -0.5), torch.float32)


@pytest.mark.gpu
def test_beyond_32_bit_offsets():
    """A memory of more than 2^32 bytes a side: the last pages are found."""
    from vectordb_amd.memory import KeyValueMemory

    page, heads, dim, pages = 64, 8, 128, 66000
    mem = KeyValueMemory(pages, page, heads, dim)
    assert mem.k.numel() > 2 ** 32
    s = Setup([100], page, heads, dim, seed=14)
    top = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda")
    k, v, q = s.randn(100, heads, dim), s.randn(100, heads, dim), s.randn(1, heads, dim)
    mem.append(k.cuda(), v.cuda(), top, ints([100]), offsets=ints([0, 100]))
    out = mem.attend(q.cuda(), top, ints([100]))
    append_ref(s.k, s.ks, k, s.table, [100], [0, 100], page)
    append_ref(s.v, s.vs, v, s.table, [100], [0, 100], page)
    check_attend(out, None, attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, [100], [0, 1], page, dim ** -0.5), torch.float32)
    assert not mem.k[:pages - 2].view(torch.uint8).any()


# ---- together ---------------------------------------------------------------------------------------------

@pytest.mark.gpu
def test_search_then_attend():
    """As it would be used: prompts appended in one go, an exact inner-product index over a head's keys finds the tokens
    that matter, attention reads those; over everything where the search returns everything."""
    from vectordb_amd import index as vi

    heads, dim, page, n = 2, 64, 16, 150
    s = Setup([n], page, heads, dim, seed=15)
    mem = s.memory()
    table, lengths = s.on_gpu()
    k, v, q = s.randn(n, heads, dim), s.randn(n, heads, dim), s.randn(1, 4 * heads, dim)
    cos, sin = angles(n, 32)
    turned = mem.append(k.cuda(), v.cuda(), table, lengths, offsets=ints([0, n]), cos=cos.cuda(), sin=sin.cuda())
    assert turned is None
    append_ref(s.k, s.ks, k, s.table, [n], [0, n], page, cos, sin)
    append_ref(s.v, s.vs, v, s.table, [n], [0, n], page)
    keys = torch.stack([turn(k[i], cos[i], sin[i], False) for i in range(n)])
    for take in (20, n + 10):
        select = torch.full((1, heads, take), -1, dtype=torch.int64, device="cuda")
        for h in range(heads):
            bf = vi.BruteforceSearch(vi.InnerProductSpace(dim), n)
            bf.add_items(keys[:, h].contiguous().numpy())
            bf.to_device(0)
            _, label = bf.search_batch(q[:, h * 4:h * 4 + 1].reshape(1, dim).contiguous().cuda(), take)
            select[0, h] = label[0]
        out, lse = mem.attend(q.cuda(), table, lengths, select=select, return_lse=True)
        check_attend(out, lse, attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, [n], [0, 1], page, dim ** -0.5, 0, select.cpu()), torch.float32)
    whole, whole_lse = mem.attend(q.cuda(), table, lengths, return_lse=True)
    ref = attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, [n], [0, 1], page, dim ** -0.5)
    check_attend(whole, whole_lse, ref, torch.float32)
    check_attend(out, lse, ref, torch.float32)  # everything was selected


@pytest.mark.gpu
def test_decoding_in_a_graph_and_on_a_stream():
    """Append and attention of one decoding step, captured once and replayed while the lengths grow; eager calls on another
    stream in between; the results are those of eager calls on a second memory, bit for bit."""
    heads, hq, dim, page, B = 2, 8, 128, 16, 3
    s = Setup([100, 100, 100], page, heads, dim, seed=16)
    a, b = s.memory(), s.memory()
    table = s.table.cuda()
    lengths = ints([5, 40, 63])
    cos, sin = (x.cuda() for x in angles(100, 64))
    k, v, q = (torch.zeros(B, h, dim, device="cuda", dtype=torch.bfloat16) for h in (heads, heads, hq))

    def step(mem, lengths):
        turned = mem.append(k, v, table, lengths, queries=q, cos=cos, sin=sin)
        return mem.attend(turned, table, lengths, return_lse=True)

    def fresh(i):
        g = torch.Generator().manual_seed(i)
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, generator=g))

    side = torch.cuda.Stream()
    fresh(0)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a, lengths)
    torch.cuda.current_stream().wait_stream(side)
    step(b, lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step(a, lengths)
    for i in range(1, 30):
        lengths += 1
        fresh(i)
        graph.replay()
        want, want_lse = step(b, lengths)
        if i % 3 == 0:
            torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8)) and torch.equal(a.v_scale, b.v_scale)


MANY = [
    # sequences, longest, most new, page, heads, q heads, dim, window: enough rows for the kernel that shares widened tokens
    (16, 150, 110, 16, 8, 16, 32, 0),
    (9, 300, 128, 64, 4, 24, 64, 0),
    (16, 140, 60, 16, 8, 32, 96, 33),
    (10, 260, 130, 32, 8, 16, 128, 0),
    (10, 200, 130, 128, 8, 16, 160, 70),
    (10, 130, 120, 16, 8, 16, 224, 0),
    (10, 150, 100, 64, 8, 16, 256, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("case", MANY, ids=lambda c: "-".join(map(str, c)))
def test_attend_many_rows(dtype, case):
    """Chunks of many sequences: of all lengths, some with no new token, an absent page, a table that is too short, NaN codes
    that only later queries see, and garbage behind the last tokens."""
    count, longest, most, page, heads, hq, dim, window = case
    t = TYPES[dtype]
    r = np.random.default_rng(dim)
    held = [longest] + [int(x) for x in r.integers(1, longest, count - 1)]
    new = [most] + [min(h, int(x)) for h, x in zip(held[1:], r.integers(0, most, count - 1))]
    s = Setup(held, page, heads, dim, seed=dim, width=-(-longest // page) - (1 if page == 16 else 0))
    s.table[1, 0] = -1
    for c in (s.k.view(torch.uint8), s.v.view(torch.uint8)):
        for b, n in enumerate(held):
            if n % page and n // page < s.table.shape[1]:
                c[s.table[b, n // page].long(), :, n % page:] = 0x7F
    for b, tok in ((0, longest - 20), (0, longest // 2), (2, held[2] - 1)):
        if tok // page < s.table.shape[1] and s.table[b, tok // page] >= 0:
            s.v.view(torch.uint8)[s.table[b, tok // page].long(), 1, tok % page, dim - 3] = 0xFF
            s.k.view(torch.uint8)[s.table[b, tok // page].long(), 2, tok % page, 1] = 0x7F
    off = offsets_of(new)
    q = s.randn(off[-1] + 2, hq, dim, dtype=t)
    mem = s.memory()
    table, lengths = s.on_gpu()
    out, lse = mem.attend(q.cuda(), table, lengths, offsets=ints(off), max_new=most, window=window, return_lse=True)
    ref = attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, off, page, dim ** -0.5, window)
    check_attend(out[:off[-1]], lse[:off[-1]], [x[:off[-1]] if torch.is_tensor(x) else x for x in ref], t)
    assert not out[off[-1]:].any()
    out = mem.attend(q.cuda(), table, lengths, offsets=ints(off), max_new=most, window=window, scale=-0.3)
    ref = attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, off, page, -0.3, window)
    check_attend(out[:off[-1]], None, [x[:off[-1]] if torch.is_tensor(x) else x for x in ref], t)


@pytest.mark.gpu
@pytest.mark.parametrize("held,window", [(199_000, 0), (199_000, 190_000), (150_000, 196_000), (199_680, 1000), (400, 180_000)])
def test_attend_long_windows(held, window):
    """A window cuts the work into other ranges than the whole table would: the workspace is the one of the call's own sizes."""
    page, heads, dim = 64, 8, 32
    s = Setup([held], page, heads, dim, seed=17, width=3120)
    q = s.randn(1, heads, dim)
    mem = s.memory()
    table, lengths = s.on_gpu()
    out, lse = mem.attend(q.cuda(), table, lengths, window=window, return_lse=True)
    check_attend(out, lse, attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, [held], [0, 1], page, dim ** -0.5, window), torch.float32)


@pytest.mark.gpu
def test_attend_long_lists():
    """More listed tokens than the table has room for: every one counts."""
    held, page, heads, dim, n = [60, 30], 16, 2, 64, 40_000
    s = Setup(held, page, heads, dim, seed=18)
    q = s.randn(2, 6, dim, dtype=torch.float16)
    select = torch.randint(-5, 70, (2, heads, n), generator=s.g)
    mem = s.memory()
    table, lengths = s.on_gpu()
    out, lse = mem.attend(q.cuda(), table, lengths, select=select.cuda(), return_lse=True)
    check_attend(out, lse, attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, [0, 1, 2], page, dim ** -0.5, 0, select), torch.float16)


def test_workspace_covers_every_range():
    """The workspace is a whole number of ranges, grows with the table and the list, and none is asked for where one range does."""
    l = _lib.lib()
    per = lambda dim: 16 * (dim + 2) * 4  # noqa: E731
    for dim in (32, 128, 256):
        for heads, group, count in ((1, 1, 1), (8, 4, 1), (8, 4, 64), (2, 20, 3)):
            m = _lib.KvMemoryStruct(16, 16, 16, 16, 10, heads, 64, dim)
            for tokens in (64, 512, 576, 4096, 200_000, 2_000_000):
                b = _lib.KvBatchStruct(16, 16, None, count, tokens // 64, count, 1)
                tiles = -(-group // 16)
                for window, select in ((0, 0), (100, 0), (190_000, 0), (0, 1), (0, 5000), (0, 3_000_000)):
                    need = l.vdb_kv_attend_workspace(m, b, heads * group, window, select)
                    seen = select or (min(tokens, window + 32) if window else tokens)
                    ranges, rest = divmod(need, count * heads * tiles * per(dim))
                    assert rest == 0 and ranges <= 384
                    if seen <= 512:
                        assert need == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim", [64, 96, 128, 224])
def test_attend_many_rows_far_scores(dtype, dim):
    """Scores of hundreds, either way, over many tiles: the softmax's reference has to move in the middle of a chunk's walk."""
    held, new, page, heads, hq = [700, 650, 70], [300, 400, 70], 16, 8, 16
    s = Setup(held, page, heads, dim, seed=18)
    t = TYPES[dtype]
    off = offsets_of(new)
    mem = s.memory()
    table, lengths = s.on_gpu()
    for mul in (60.0, -60.0, 0.0):
        q = s.randn(off[-1], hq, dim, dtype=t) * mul
        out, lse = mem.attend(q.cuda(), table, lengths, offsets=ints(off), max_new=max(new), return_lse=True)
        check_attend(out, lse, attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, off, page, dim ** -0.5), t)


@pytest.mark.gpu
@pytest.mark.parametrize("count,most", [(64, 40), (65, 40), (130, 70)])
def test_attend_many_sequences(count, most):
    """Up to and beyond the 64 sequences whose work is put in order: every row is written, whatever the lengths, also with none
    held, fewer held than new, none new; and whatever the caller says is the longest chunk."""
    page, heads, hq, dim = 16, 2, 8, 64
    r = np.random.default_rng(count)
    held = [int(x) for x in r.integers(0, 120, count)]
    new = [int(x) for x in r.integers(0, most + 1, count)]
    held[3], new[3], held[4], new[4], new[5], held[6], new[6] = 5, most, 0, 2, 0, 119, most
    s = Setup(held, page, heads, dim, seed=count)
    off = offsets_of(new)
    q = s.randn(off[-1], hq, dim, dtype=torch.bfloat16)
    mem = s.memory()
    table, lengths = s.on_gpu()
    ref = attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, off, page, dim ** -0.5, 50)
    for said in (most, 16, 100_000):
        out, lse = mem.attend(q.cuda(), table, lengths, offsets=ints(off), max_new=said, window=50, return_lse=True)
        check_attend(out, lse, ref, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("held,new", [([2100], [2048]), ([513] * 4, [512] * 4), ([5000, 64, 65, 2000], [30, 64, 1, 900])])
def test_attend_many_rows_every_item(held, new):
    """Work in the order of its cost, over sequences that are equal, alone or very different: nothing is left out or done twice."""
    page, heads, hq, dim = 64, 8, 32, 32
    s = Setup(held, page, heads, dim, seed=19)
    off = offsets_of(new)
    q = s.randn(off[-1], hq, dim, dtype=torch.bfloat16)
    mem = s.memory()
    table, lengths = s.on_gpu()
    out, lse = mem.attend(q.cuda(), table, lengths, offsets=ints(off), max_new=max(new), return_lse=True)
    check_attend(out, lse, attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, off, page, dim ** -0.5), torch.bfloat16)


@pytest.mark.gpu
def test_rows_with_odd_strides_of_single_dimensions():
    """One token or one head out of something larger: a stride that nobody steps along may be any number."""
    page, dim = 16, 32
    for tokens, heads in ((1, 2), (3, 1), (1, 1)):
        s = Setup([20] * tokens, page, heads, dim, seed=20)
        mem = s.memory()
        table, lengths = s.on_gpu()
        k, v, q = s.randn(tokens, heads, dim), s.randn(tokens, heads, dim), s.randn(tokens, heads, dim)
        def odd(x):
            return x.cuda().as_strided(x.shape, (heads * dim if tokens > 1 else 5, dim if heads > 1 else 3, 1))
        mem.append(odd(k), odd(v), table, lengths)
        off = list(range(tokens + 1))
        append_ref(s.k, s.ks, k, s.table, s.lengths, off, page)
        append_ref(s.v, s.vs, v, s.table, s.lengths, off, page)
        assert same_codes(mem.k, s.k) and same_codes(mem.v, s.v)
        out = mem.attend(odd(q), table, lengths)
        check_attend(out, None, attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, s.lengths, off, page, dim ** -0.5), torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("new", [[1, 1], [200, 256]])
def test_attend_scales_far_apart(dtype, new):
    """Pages of zeros (whose scale is the smallest that is stored), of ordinary and of huge values in one sequence: the zeros
    count in the softmax's sum as anything else does."""
    held, page, heads, hq, dim = [520, 300], 16, 16, 32, 64
    t = TYPES[dtype]
    s = Setup(held, page, heads, dim, seed=21)
    for b in range(2):
        for p in range(-(-held[b] // page)):
            i = s.table[b, p].long()
            if (p // 5) % 3 == 0:
                s.v.view(torch.uint8)[i] = 0
                s.vs[i] = 2.0 ** -100
            else:
                s.vs[i] = 2.0 ** (-2 if (p // 5) % 3 == 1 or dtype == "f16" else 40)
    off = offsets_of(new)
    q = s.randn(off[-1], hq, dim, dtype=t)
    mem = s.memory()
    table, lengths = s.on_gpu()
    out, lse = mem.attend(q.cuda(), table, lengths, offsets=None if max(new) == 1 else ints(off), max_new=max(new), return_lse=True)
    check_attend(out, lse, attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, off, page, dim ** -0.5), t)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim", [("f32", 64), ("bf16", 128), ("f32", 192)])
@pytest.mark.parametrize("count,heads,n", [(19, 2, 70), (8, 3, 2500), (130, 4, 40)])
def test_attend_selected_batches(dtype, dim, count, heads, n):
    """More sequences than dies, and a rest; lists in one range and in several; few rows and many."""
    page, hq = 16, 2 * heads
    r = np.random.default_rng(n)
    held = [int(x) for x in r.integers(0, 200, count)]
    s = Setup(held, page, heads, dim, seed=n)
    q = s.randn(count, hq, dim, dtype=TYPES[dtype])
    select = torch.randint(-5, 220, (count, heads, n), generator=s.g)
    mem = s.memory()
    table, lengths = s.on_gpu()
    out, lse = mem.attend(q.cuda(), table, lengths, select=select.cuda(), return_lse=True)
    check_attend(out, lse, attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, list(range(count + 1)), page, dim ** -0.5, 0, select), TYPES[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["chunks", "many", "selected", "ranges"])
def test_attend_captured_and_on_two_streams(kind):
    """Each way of attention captured once and replayed with other lengths, eager calls in between on two streams at a time: every
    result is, bit for bit, that of the same call alone."""
    page, heads, hq, dim = 16, 8, 32, 64
    new = dict(chunks=[20, 7], many=[300, 200], selected=[1, 1], ranges=[1, 1])[kind]
    s = Setup([1900, 1400], page, heads, dim, seed=22)
    off = offsets_of(new)
    mem = s.memory()
    table, lengths = s.on_gpu()
    offsets = None if max(new) == 1 else ints(off)
    select = torch.randint(-3, 2000, (2, heads, 3000), generator=s.g).cuda() if kind == "selected" else None
    q = s.randn(off[-1], hq, dim, dtype=torch.bfloat16).cuda()

    def step(lengths):
        return mem.attend(q, table, lengths, offsets=offsets, max_new=max(new), select=select, return_lse=True)

    held = [[1900, 1400], [600, 1399], [350, 230], [1, 1000], [0, 0], [1700, 320]]
    alone = [step(ints(h)) for h in held]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(lengths)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(lengths)
    other = [ints(h) for h in held]
    torch.cuda.synchronize()
    for turn_ in range(2):
        for i, h in enumerate(held):
            lengths.copy_(other[i])
            graph.replay()
            with torch.cuda.stream(side):
                b = [step(x) for x in other]
            a = [step(x) for x in other]
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, alone[i]))
            for results in (a, b):
                assert all(torch.equal(x, y) for r, w in zip(results, alone) for x, y in zip(r, w))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,held", [(32, [8000, 5, 3100]), (96, [9000, 513]), (160, [7900]), (256, [9100, 4096, 0]), (64, [40_000, 700, 1])])
def test_attend_ranges_joined(dtype, dim, held):
    """One token over so much that its tokens are cut into up to 16 ranges, or more: their joints, for each way of joining."""
    page, heads, hq = 64, 2, 6
    s = Setup(held, page, heads, dim, seed=dim)
    q = s.randn(len(held), hq, dim, dtype=TYPES[dtype]) * 3
    mem = s.memory()
    table, lengths = s.on_gpu()
    out, lse = mem.attend(q.cuda(), table, lengths, return_lse=True)
    ref = attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, list(range(len(held) + 1)), page, dim ** -0.5)
    check_attend(out, lse, ref, TYPES[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,interleaved", [("f32", False), ("bf16", True), ("f16", False)])
def test_append_many_large_pages(dtype, interleaved):
    """So many pages that keys and values are stored by launches of their own, with and without queries, turned and not."""
    held, new, page, heads, dim, hq = [1100] * 8, [1000] * 8, 128, 32, 32, 32
    off = offsets_of(new)
    k, v, q = (Setup([1], 16, 1, 32, seed=23 + i).randn(off[-1], heads, dim, dtype=TYPES[dtype]) for i in range(3))
    cos, sin = angles(1100, 16)
    for rot in (True, False):
        s = Setup(held, page, heads, dim, seed=24)
        mem = s.memory()
        table, lengths = s.on_gpu()
        angle = dict(cos=cos.cuda(), sin=sin.cuda(), interleaved=interleaved) if rot else {}
        got = mem.append(k.cuda(), v.cuda(), table, lengths, offsets=ints(off), max_new=1000, queries=q.cuda() if rot else None, **angle)
        whole = s.memory()  # the same, one sequence a call
        for b in range(8):
            rows = slice(off[b], off[b + 1])
            one = whole.append(k[rows].cuda(), v[rows].cuda(), table[b:b + 1], lengths[b:b + 1], offsets=ints([0, 1000]), max_new=1000,
                               queries=q[rows].cuda() if rot else None, **angle)
            assert not rot or torch.equal(one, got[rows])
        assert same_codes(mem.k, whole.k.cpu()) and same_codes(mem.v, whole.v.cpu())
        assert torch.equal(mem.k_scale, whole.k_scale) and torch.equal(mem.v_scale, whole.v_scale)
        for b in (0, 7):  # and one of them by the formula
            rows = slice(off[b], off[b + 1])
            ref = Setup(held, page, heads, dim, seed=24)
            append_ref(ref.k, ref.ks, k[rows], ref.table[b:b + 1], held[b:b + 1], [0, 1000], page, *((cos, sin, interleaved) if rot else ()))
            append_ref(ref.v, ref.vs, v[rows], ref.table[b:b + 1], held[b:b + 1], [0, 1000], page)
            at = ref.table[b][ref.table[b] >= 0].long()
            assert same_codes(mem.k[at.cuda()], ref.k[at]) and same_codes(mem.v[at.cuda()], ref.v[at])


@pytest.mark.parametrize("count,tokens,offsets", [(0, 0, None), (0, 0, 16), (0, 5, 16), (3, 0, 16)])
def test_nothing_to_attend_to_without_a_device(count, tokens, offsets):
    """No sequences, or no new rows: no workspace and no work, for every way of attention."""
    l = _lib.lib()
    for heads, group, width, most in ((1, 1, 1, 0), (8, 4, 1000, 0), (8, 4, 1000, 2048), (2, 20, 100_000, 1)):
        m = _lib.KvMemoryStruct(16, 16, 16, 16, 10, heads, 64, 128)
        b = _lib.KvBatchStruct(16, 16, offsets, count, width, tokens, most)
        for window, select in ((0, 0), (700, 0), (0, 5000)):
            if select and offsets:
                continue
            assert l.vdb_kv_attend_workspace(m, b, heads * group, window, select) == 0
            assert l.vdb_kv_attend_device(m, b, 0, None, 128, 64, heads * group, 1.0, window, 16 if select else None, select, None, None, None, 0, None) == _lib.VDB_OK


@pytest.mark.gpu
def test_nothing_to_attend_to():
    """The same from Python: empty results of the right shape, zeros for rows of no sequence."""
    s = Setup([40, 70], 16, 2, 64, seed=24)
    mem = s.memory()
    table, lengths = s.on_gpu()
    q = s.randn(5, 4, 64).cuda()
    out, lse = mem.attend(q[:0], table, lengths, offsets=ints([0, 0, 0]), return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    out, lse = mem.attend(q[:0], table[:0], lengths[:0], return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    assert mem.attend(q[:0], table[:0], lengths[:0], select=torch.zeros((0, 2, 7), dtype=torch.int64, device="cuda")).shape == (0, 4, 64)
    assert not mem.attend(q, table[:0], lengths[:0], offsets=ints([0])).any()
    mem.append(q[:0, :2], q[:0, :2], table, lengths, offsets=ints([0, 0, 0]))
    assert same_codes(mem.k, s.k)


UNDERSTATED = [
    # held, new, heads, q heads, dim, window: tokens in ranges, and more new ones than the caller says
    ([4000], [3], 2, 8, 64, 0),
    ([8000, 300], [16, 20], 1, 1, 32, 0),
    ([40_000, 1000], [9, 30], 1, 2, 128, 0),  # more than 16 ranges
    ([3009], [16], 1, 1, 64, 2016),           # a window just short of a whole number of ranges, which a tile's rows pass
    ([1500, 5000], [16, 33], 1, 1, 96, 992),
    ([40_000], [24], 1, 1, 32, 16_368),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("case", UNDERSTATED, ids=lambda c: "-".join(map(str, c[0] + c[1] + list(c[2:]))))
def test_attend_understated_max_new(dtype, case):
    """A wrong max_new costs time only: every row of a tile whose tokens are cut into ranges is joined."""
    held, new, heads, hq, dim, window = case
    page = 64
    s = Setup(held, page, heads, dim, seed=25)
    off = offsets_of(new)
    q = s.randn(off[-1], hq, dim, dtype=TYPES[dtype])
    mem = s.memory()
    table, lengths = s.on_gpu()
    ref = attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, off, page, dim ** -0.5, window)
    for said in (1, 2, max(new)):
        out, lse = mem.attend(q.cuda(), table, lengths, offsets=ints(off), max_new=said, window=window, return_lse=True)
        check_attend(out, lse, ref, TYPES[dtype])


@pytest.mark.gpu
def test_attend_replayed_with_other_offsets():
    """A step captured for one or two new tokens a sequence is replayed for other numbers of them, into the same buffers."""
    page, heads, hq, dim, held = 64, 1, 2, 64, [4000, 2900]
    s = Setup(held, page, heads, dim, seed=26)
    mem = s.memory()
    table, lengths = s.on_gpu()
    q = s.randn(30, hq, dim, dtype=torch.float16).cuda()
    offsets = ints([0, 1, 3])

    def step():
        return mem.attend(q, table, lengths, offsets=offsets, max_new=2, return_lse=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    for off in ([0, 1, 3], [0, 16, 30], [2, 2, 19], [0, 30, 30], [0, 1, 3]):
        offsets.copy_(ints(off))
        graph.replay()
        want, want_lse = step()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        ref = attend_ref(q.cpu(), s.k, s.v, s.ks, s.vs, s.table, held, off, page, dim ** -0.5)
        rows = slice(off[0], off[2])
        check_attend(out[rows], lse[rows], [x[rows] if torch.is_tensor(x) else x for x in ref], torch.float16)
        assert not out[:off[0]].any() and not out[off[2]:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim", [32, 128, 224])
def test_attend_scales_of_pages_left_behind(dtype, dim):
    """Pages that the window has left behind may hold anything, scales included, also where a tile of tokens begins in one."""
    held, new, page, heads, hq, window = [600, 533, 330], [400, 350, 328], 16, 8, 16, 40
    s = Setup(held, page, heads, dim, seed=27)
    off = offsets_of(new)
    for b in range(3):
        for p in range(max(0, held[b] - new[b] - window + 1) // page):
            i = s.table[b, p].long()
            s.ks[i], s.vs[i] = float("-inf"), (float("inf"), float("nan"), 2.0 ** 127)[p % 3]
    q = s.randn(off[-1], hq, dim, dtype=TYPES[dtype])
    mem = s.memory()
    table, lengths = s.on_gpu()
    out, lse = mem.attend(q.cuda(), table, lengths, offsets=ints(off), max_new=max(new), window=window, return_lse=True)
    check_attend(out, lse, attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, off, page, dim ** -0.5, window), TYPES[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim", [32, 64, 160, 256])
@pytest.mark.parametrize("group", [1, 16, 17])
def test_attend_selected_blocks_of_eight_waves(dtype, dim, group):
    """Few rows of selected tokens: the waves' parts of one, sixteen and seventeen rows are joined by the threads that have a row."""
    held, page, heads, n = [90, 0, 300], 16, 2, 333
    s = Setup(held, page, heads, dim, seed=28)
    q = s.randn(3, heads * group, dim, dtype=TYPES[dtype])
    select = torch.randint(-5, 310, (3, heads, n), generator=s.g)
    mem = s.memory()
    table, lengths = s.on_gpu()
    out, lse = mem.attend(q.cuda(), table, lengths, select=select.cuda(), return_lse=True)
    check_attend(out, lse, attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, [0, 1, 2, 3], page, dim ** -0.5, 0, select), TYPES[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens,hq,interleaved", [(5, 4, False), (1, 1, True), (700, 96, False), (700, 96, True)])
def test_append_queries_of_no_sequence(dtype, tokens, hq, interleaved):
    """No sequences, but rows: the queries are copied, few of them and many, whatever their strides."""
    s = Setup([20], 16, 2, 64, seed=29)
    mem = s.memory()
    cos, sin = (x.cuda() for x in angles(30, 16))
    k = s.randn(tokens, 2, 64, dtype=TYPES[dtype]).cuda()
    fused = s.randn(tokens, hq + 3, 64, dtype=TYPES[dtype]).cuda()
    q = fused[:, 2:2 + hq]
    got = mem.append(k, k, ints([]).view(0, 2), ints([]), offsets=ints([0]), queries=q, cos=cos, sin=sin, interleaved=interleaved)
    assert torch.equal(got, q)
    assert same_codes(mem.k, s.k) and torch.equal(mem.k_scale.cpu(), s.ks)
    assert mem.append(k, k, ints([]).view(0, 2), ints([]), offsets=ints([0])) is None


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("new", [[1, 1], [20, 3]])
def test_append_angles_of_no_position(new, interleaved):
    """Tables of angles without rows: no key is stored, every value is, and every query is not a number."""
    held, page, heads, dim = [40, 25], 16, 2, 64
    s = Setup(held, page, heads, dim, seed=30)
    mem = s.memory()
    table, lengths = s.on_gpu()
    off = offsets_of(new)
    k, v, q = (s.randn(off[-1], h, dim, dtype=torch.bfloat16) for h in (heads, heads, 4))
    none = torch.zeros((0, 16), device="cuda")
    got = mem.append(k.cuda(), v.cuda(), table, lengths, offsets=None if max(new) == 1 else ints(off), queries=q.cuda(), cos=none, sin=none, interleaved=interleaved)
    append_ref(s.v, s.vs, v, s.table, held, off, page)
    assert same_codes(mem.k, s.k) and torch.equal(mem.k_scale.cpu(), s.ks)
    assert same_codes(mem.v, s.v) and torch.equal(mem.v_scale.cpu(), s.vs)
    assert torch.isnan(got).all()


@pytest.mark.gpu
@pytest.mark.parametrize("count,heads,longest,page,dim", [(1000, 64, 300, 64, 64), (300, 8, 2000, 16, 32), (65_535, 2, 1, 16, 32)])
def test_append_without_max_new(count, heads, longest, page, dim):
    """Many sequences and no word about the longest: the launch stays within bounds (1000 x 128 x 67 blocks of 512 threads would be
    2^32 of them), and every token is stored."""
    from vectordb_amd.memory import KeyValueMemory

    r = np.random.default_rng(count)
    new = [int(x) for x in r.integers(0, 9, count)]
    new[count // 2] = longest
    held = [n + int(x) for n, x in zip(new, r.integers(0, 30, count))]
    off = offsets_of(new) if count < 10_000 else [0] + list(np.cumsum(new))
    assert count != 1000 or 128 * 1000 * 512 * ((off[-1] + 2 * page - 2) // page) >= 2 ** 32
    need = np.array([-(-h // page) for h in held])
    at = np.cumsum(need) - need
    width = max(int(need.max()), off[-1] // page + 2 if count < 10_000 else 0)
    wide = np.arange(width)
    table = torch.from_numpy(np.where(wide < need[:, None], at[:, None] + wide, -1).astype(np.int32)).cuda()
    g = torch.Generator(device="cuda").manual_seed(count)
    k, v = (torch.randn(off[-1], heads, dim, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    pages = int(need.sum())
    a, b = KeyValueMemory(pages, page, heads, dim), KeyValueMemory(pages, page, heads, dim)
    a.append(k, v, table, ints(held), offsets=ints(off))
    b.append(k, v, table, ints(held), offsets=ints(off), max_new=max(new))
    for x, y in ((a.k, b.k), (a.v, b.v)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert torch.equal(a.k_scale, b.k_scale) and torch.equal(a.v_scale, b.v_scale)
    i = count // 2  # and the longest by the formula
    ids = table[i, :need[i]].long()
    ks, ref, here = torch.ones(len(ids), heads), torch.zeros(len(ids), heads, page, dim).to(E4M3), torch.arange(len(ids), dtype=torch.int32)[None]
    append_ref(ref, ks, k[off[i]:off[i + 1]].cpu(), here, [held[i]], [0, new[i]], page)
    assert same_codes(a.k[ids], ref) and torch.equal(a.k_scale[ids].cpu(), ks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,page,dim,interleaved", [("f32", 16, 32, False), ("bf16", 64, 96, True), ("f16", 32, 64, False), ("bf16", 128, 64, False)])
def test_append_one_long_among_short(dtype, page, dim, interleaved):
    """One prompt among many short ones or none, with and without a word about the longest: pages absent, positions below 0 and
    without angles, rows of no sequence, a last sequence that claims rows which are not there."""
    heads, hq, count, t = 2, 3, 70, TYPES[dtype]
    r = np.random.default_rng(page)
    new = [int(x) for x in r.integers(0, 3, count)]
    new[0], new[31], new[68] = 0, 17 * page + 5, page
    held = [n + int(x) for n, x in zip(new, r.integers(0, 20, count))]
    held[5], new[5], held[68], new[69] = 2, 6, page - 3, 2
    s = Setup(held, page, heads, dim, seed=31, width=-(-max(held) // page))
    s.table[31, 3], s.table[31, 7] = -1, s.ks.shape[0]
    off = [n + 3 for n in offsets_of(new)]
    total = off[-1] + 4
    off[-1] += 9  # beyond the rows that there are
    k, v, q = s.randn(total, heads, dim, dtype=t), s.randn(total, heads, dim, dtype=t), s.randn(total, hq, dim, dtype=t)
    cos, sin = angles(max(held) - 11, 16)
    first = Setup(held, page, heads, dim, seed=31, width=-(-max(held) // page))
    append_ref(s.k, s.ks, k, s.table, held, off, page, cos, sin, interleaved)
    append_ref(s.v, s.vs, v, s.table, held, off, page)
    want = q.clone()
    for b in range(count - 1):
        for i in range(new[b]):
            pos = held[b] - new[b] + i
            want[off[b] + i] = turn(q[off[b] + i].float(), cos[pos], sin[pos], interleaved).to(t) if 0 <= pos < cos.shape[0] else torch.full_like(q[0], float("nan"))
    for said in (None, max(new), 1):
        mem = first.memory()
        table, lengths = s.on_gpu()
        got = mem.append(k.cuda(), v.cuda(), table, lengths, offsets=ints(off), max_new=said, queries=q.cuda(), cos=cos.cuda(), sin=sin.cuda(), interleaved=interleaved)
        assert same_codes(mem.k, s.k) and same_codes(mem.v, s.v)
        assert torch.equal(mem.k_scale.cpu(), s.ks) and torch.equal(mem.v_scale.cpu(), s.vs)
        assert same_codes(got, want.float())


def test_append_too_many_blocks_without_a_device():
    """So many sequences and heads that one launch cannot have the threads: refused, not cut off."""
    l = _lib.lib()
    m = _lib.KvMemoryStruct(16, 16, 16, 16, 10, 100, 64, 256)
    b = _lib.KvBatchStruct(16, 16, 16, 65_535, 4, 1 << 20, 64)
    assert l.vdb_kv_append_device(m, b, 0, 16, 25_600, 256, 16, 25_600, 256, None, None, 0, 0, 0, None, 0, 0, 0, None, None) == _lib.VDB_ERR_INVALID
    assert "too many" in l.vdb_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim", [("f32", 32), ("bf16", 128), ("f16", 64)])
def test_attend_one_long_among_short(dtype, dim):
    """One prompt among many short ones or none, with and without a word about the longest; rows of no sequence before, and a last
    sequence that claims rows which are not there."""
    page, heads, hq, count, t = 16, 2, 8, 90, TYPES[dtype]
    r = np.random.default_rng(dim)
    new = [int(x) for x in r.integers(0, 4, count)]
    new[0], new[40], new[88], new[89] = 0, 600, 70, 2
    held = [n + int(x) for n, x in zip(new, r.integers(0, 50, count))]
    held[5], new[5] = 3, 9
    s = Setup(held, page, heads, dim, seed=32)
    off = [n + 5 for n in offsets_of(new)]
    total = off[-1]
    off[-1] += 2
    q = s.randn(total, hq, dim, dtype=t)
    mem = s.memory()
    table, lengths = s.on_gpu()
    ref = attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, off, page, dim ** -0.5)
    for said in (None, max(new), 70):
        out, lse = mem.attend(q.cuda(), table, lengths, offsets=ints(off), max_new=said, return_lse=True)
        rows = slice(off[0], off[-2])
        check_attend(out[rows], lse[rows], [x[rows] if torch.is_tensor(x) else x for x in ref], t)
        assert not out[:off[0]].any() and not out[off[-2]:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [32, 96, 128, 256])
@pytest.mark.parametrize("kind", ["single", "chunks", "selected", "ranges"])
def test_attend_bf16_results_are_rounded_once(kind, dim):
    """Weights take part with 16 bits at least (two bf16 parts, each rounded: 2^-16 of each): a bf16 result is off by its own half
    step, 2^-8 of it, and by what f32 sums leave, but not by 2^-8 of all that it was added up from."""
    page, heads, hq, t = 16, 2, 6, torch.bfloat16
    held, new = dict(single=([3, 20, 300], [1, 1, 1]), chunks=([4, 70], [3, 9]), selected=([300, 40], [1, 1]), ranges=([2500], [1]))[kind]
    s = Setup(held, page, heads, dim, seed=33)
    off = offsets_of(new)
    q = s.randn(off[-1], hq, dim, dtype=t)
    select = torch.randint(-1, 300, (2, heads, 11), generator=s.g) if kind == "selected" else None
    mem = s.memory()
    table, lengths = s.on_gpu()
    got = mem.attend(q.cuda(), table, lengths, offsets=None if max(new) == 1 else ints(off), max_new=max(new), select=None if select is None else select.cuda())
    out, _, mass, size, n = attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, off, page, dim ** -0.5, 0, select)
    score, many = (3 * dim + 16) * EPS * size, (n / 32 + 64) * EPS
    tol = (2 * score[..., None] + 2.0 ** -16 + 2 * many) * mass * 1.01 + 2.0 ** -8 * 1.01 * out.abs() + 1e-38
    assert ((got.double().cpu() - out).abs() <= tol).all()


@pytest.mark.gpu
def test_gradients_are_refused():
    """A tensor that requires a gradient: refused where torch records operations, taken where it does not."""
    from vectordb_amd.memory import KeyValueMemory
    from vectordb_amd.rows4 import Rows4

    s = Setup([5, 20], 16, 2, 64, seed=34)
    mem = s.memory()
    table, lengths = s.on_gpu()
    cos, sin = (x.cuda() for x in angles(30, 16))
    kv, q, x = s.randn(2, 2, 64).cuda(), s.randn(2, 4, 64).cuda(), s.randn(3, 40).cuda()
    rows = Rows4.pack(x)
    grad = lambda t: t.clone().requires_grad_()  # noqa: E731
    for call in [lambda f: mem.attend(f(q), table, lengths), lambda f: mem.append(f(kv), kv, table, lengths), lambda f: mem.append(kv, f(kv), table, lengths),
                 lambda f: mem.append(kv, kv, table, lengths, queries=f(q), cos=cos, sin=sin), lambda f: mem.append(kv, kv, table, lengths, queries=f(q)),
                 lambda f: mem.append(kv, kv, table, lengths, cos=f(cos), sin=sin), lambda f: rows.products(x, out=f(torch.zeros(3, 3, device="cuda"))),
                 lambda f: rows.products(f(x)), lambda f: rows.products(f(x)[0]), lambda f: Rows4.pack(f(x)).codes,
                 lambda f: KeyValueMemory.from_tensors(mem.k, mem.v, f(mem.k_scale), mem.v_scale).attend(q, table, lengths)]:
        with pytest.raises(ValueError, match="gradient"):
            call(grad)
        with torch.no_grad():
            a = call(grad)
        b = call(lambda t: t)
        assert (a is None and b is None) or torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("count,heads,group,dim", [(130, 1, 64, 32), (70, 2, 200, 64), (40, 4, 70, 128)])
def test_attend_one_token_of_many_heads(dtype, count, heads, group, dim):
    """One new token a sequence, without offsets, but so many query heads a key head that the kernel for many rows takes them, up to
    and beyond the 64 sequences whose work it puts in order."""
    page = 16
    r = np.random.default_rng(count)
    held = [int(x) for x in r.integers(0, 150, count)]
    s = Setup(held, page, heads, dim, seed=35)
    q = s.randn(count, heads * group, dim, dtype=TYPES[dtype])
    mem = s.memory()
    table, lengths = s.on_gpu()
    for window in (0, 30):
        out, lse = mem.attend(q.cuda(), table, lengths, window=window, return_lse=True)
        ref = attend_ref(q, s.k, s.v, s.ks, s.vs, s.table, held, list(range(count + 1)), page, dim ** -0.5, window)
        check_attend(out, lse, ref, TYPES[dtype])
