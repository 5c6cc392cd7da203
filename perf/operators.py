"""Cases and plain forms of the operators on rows held in few bits: products with 4-bit rows, the append to an 8-bit
key / value memory with the position rotation applied on the way, and the attention that reads that memory.

``run`` computes a case with elementary torch operations, or, where ``own`` is true, through the package."""
from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
DEVICE = "cuda"


def listed():
    return [
        # one query against the 10 000 x 128 rows of the smallest configuration: all latency
        dict(name="products_10k_128_q1", op="products", n=10_000, dim=128, nq=1, dtype="f32"),
        # one query against the million 960-dimensional rows of the brute-force configuration: the bytes of the rows
        dict(name="products_1m_960_q1", op="products", n=1_000_000, dim=960, nq=1, dtype="f32"),
        # a few queries of an encoder in bf16 against a million 128-dimensional rows: the output weighs as much as the rows
        dict(name="products_1m_128_q16", op="products", n=1_000_000, dim=128, nq=16, dtype="bf16"),
        # odd sizes: a last group of 4 columns, a last tile of rows that is not full
        dict(name="products_250k_100_q7", op="products", n=250_001, dim=100, nq=7, dtype="f16"),
        # a decoding step of 64 sequences: one token each, queries rotated beside the keys
        dict(name="append_64x1", op="append", batch=64, new_max=1, past=4096, page=64, hq=32, hkv=8, dim=128, rot=128, dtype="bf16", even=True),
        # prompts of different lengths in f32, half of the dimensions rotated, pages of 16 tokens
        dict(name="append_5x700_f32", op="append", batch=5, new_max=700, past=333, page=16, hq=12, hkv=12, dim=96, rot=48, dtype="f32", even=False),
        # long prompts: the copy's bytes
        dict(name="append_8x8192", op="append", batch=8, new_max=8192, past=0, page=128, hq=32, hkv=8, dim=128, rot=128, dtype="bf16", even=True),
        # one short sequence: the latency of a step
        dict(name="attend_1x500", op="attend", batch=1, new_max=1, len_max=500, page=16, hq=8, hkv=8, dim=64, window=0, select=0, dtype="f16", even=True),
        # a decoding step of 64 sequences of different lengths
        dict(name="attend_64x8192", op="attend", batch=64, new_max=1, len_max=8192, page=64, hq=32, hkv=8, dim=128, window=0, select=0, dtype="bf16", even=False),
        # two very long sequences: the work has to be split over the keys
        dict(name="attend_2x500k", op="attend", batch=2, new_max=1, len_max=500_003, page=64, hq=16, hkv=2, dim=128, window=0, select=0, dtype="f16", even=True),
        # chunks of prompts over what the memory holds already: matrix products
        dict(name="attend_chunk_4x2048", op="attend", batch=4, new_max=2048, len_max=6000, page=64, hq=32, hkv=8, dim=128, window=0, select=0, dtype="bf16", even=False),
        # the 2048 tokens that a search returned for each sequence and head, out of a memory beyond 32-bit offsets, in f32
        dict(name="attend_select_32x2048", op="attend", batch=32, new_max=1, len_max=131_072, page=64, hq=32, hkv=8, dim=128, window=0, select=2048, dtype="f32", even=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["products", "append", "attend"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "products":
        dim = _log(rng, 8, 2000)
        return dict(op=op, n=_log(rng, 1000, max(1001, min(1_000_000, 900_000_000 // dim))), dim=dim, nq=_log(rng, 1, 16), dtype=dtype)
    hkv = rng.choice([1, 2, 3, 4, 8])
    hq = hkv * rng.choice([1, 2, 4, 5, 8])
    dim = rng.choice([32, 64, 96, 128, 160, 256])
    page = rng.choice([16, 32, 64, 128])
    even = rng.random() < 0.3
    if op == "append":
        batch = _log(rng, 1, 64)
        new_max = 1 if rng.random() < 0.4 else _log(rng, 2, max(3, 40_000_000 // (batch * (hq + 2 * hkv) * dim)))
        return dict(op=op, batch=batch, new_max=min(new_max, 8192), past=rng.choice([0, _log(rng, 1, 4000)]), page=page, hq=hq, hkv=hkv, dim=dim,
                    rot=rng.choice([0, 32, dim]), dtype=dtype, even=even)
    kind = rng.choice(["token", "token", "chunk", "select"])
    window = rng.choice([0, 0, _log(rng, 1, 5000)])
    if kind == "chunk":
        batch, len_max = rng.randint(1, 4), _log(rng, 20, 5000)
        return dict(op=op, batch=batch, new_max=min(len_max, _log(rng, 2, 1500)), len_max=len_max, page=page, hq=hq, hkv=hkv, dim=dim, window=window,
                    select=0, dtype=dtype, even=even)
    batch = _log(rng, 1, 64)
    len_max = _log(rng, 1, min(300_000, 250_000_000 // (batch * hkv * dim)))
    select = 0 if kind == "token" else _log(rng, 1, min(2048, len_max))
    return dict(op=op, batch=batch, new_max=1, len_max=len_max, page=page, hq=hq, hkv=hkv, dim=dim, window=0 if select else window, select=select, dtype=dtype, even=even)


def _lengths(case):
    """(tokens held after the call, tokens that the call brings) of each sequence: a property of the case."""
    r = random.Random("%s-%d-%d-%d" % (case["op"], case["batch"], case["new_max"], case["page"]))
    if case["op"] == "append":
        new = [case["new_max"] if case["even"] else r.randint(max(1, case["new_max"] // 3), case["new_max"]) for _ in range(case["batch"])]
        past = [case["past"] if case["even"] else r.randint(0, case["past"]) for _ in range(case["batch"])]
        return [p + n for p, n in zip(past, new)], new
    held = [case["len_max"] if case["even"] or i == 0 else r.randint(max(1, case["len_max"] // 8), case["len_max"]) for i in range(case["batch"])]
    new = [min(h, case["new_max"] if case["even"] or i == 0 else r.randint(1, case["new_max"])) for i, h in enumerate(held)]
    return held, new


def _codes(shape, g):
    """e4m3 codes of normally distributed values that fill the type's range as a page's scale makes them do."""
    total = math.prod(shape)
    base = (torch.randn(min(total, 16_000_057), generator=g, device=DEVICE) * 90).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return base.repeat(-(-total // base.numel()))[:total].reshape(shape).view(torch.float8_e4m3fn)


def _memory(case, held, g, dim, hkv, page):
    need = [-(-h // page) for h in held]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEVICE).int()
    at = torch.tensor([sum(need[:i]) for i in range(len(need))], device=DEVICE)
    table = order[(at[:, None] + torch.arange(max(need), device=DEVICE)[None, :]).clamp_(max=pages - 1)]
    scale = lambda: torch.exp2(torch.randint(-8, -5, (pages, hkv), generator=g, device=DEVICE).float())  # noqa: E731
    return dict(k=_codes((pages, hkv, page, dim), g), v=_codes((pages, hkv, page, dim), g), k_scale=scale(), v_scale=scale(),
                table=table.contiguous(), lengths=torch.tensor(held, dtype=torch.int32, device=DEVICE))


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    t = TYPES[case["dtype"]]
    rand = lambda *shape: torch.randn(shape, generator=g, device=DEVICE).to(t)  # noqa: E731
    s = dict(case=case)
    if case["op"] == "products":
        groups = -(-case["dim"] // 32)
        s["codes"] = torch.randint(0, 256, (case["n"], groups * 16), generator=g, device=DEVICE, dtype=torch.uint8)
        s["codes"].view(case["n"], groups * 16)[:, (case["dim"] + 1) // 2:] = 0
        if case["dim"] % 2:
            s["codes"][:, case["dim"] // 2] &= 15
        s["scales"] = torch.randint(121, 127, (case["n"], groups), generator=g, device=DEVICE, dtype=torch.uint8)
        s["x"] = rand(case["nq"], case["dim"])
        return s
    held, new = _lengths(case)
    s |= _memory(case, held, g, case["dim"], case["hkv"], case["page"])
    total = sum(new)
    s["q"] = rand(total, case["hq"], case["dim"])
    s["offsets"] = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEVICE) if case["new_max"] > 1 else None
    if case["op"] == "append":
        s["new_k"], s["new_v"] = rand(total, case["hkv"], case["dim"]), rand(total, case["hkv"], case["dim"])
        s["cos"] = s["sin"] = None
        if case["rot"]:
            angle = torch.arange(max(held), device=DEVICE, dtype=torch.float64)[:, None] * 10000.0 ** (
                -torch.arange(0, case["rot"], 2, device=DEVICE, dtype=torch.float64) / case["rot"])
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    elif case["select"]:
        s["select"] = torch.randint(0, case["len_max"], (case["batch"], case["hkv"], case["select"]), generator=g, device=DEVICE)
        s["select"] = torch.where(s["select"] < s["lengths"][:, None, None], s["select"], -1)
        s["select"][:, :, 0] = 0
    return s


# ---- plain forms ------------------------------------------------------------------------------

def _plain_products(s):
    case = s["case"]
    one = torch.tensor(E2M1 + [-v for v in E2M1], device=DEVICE)
    both = torch.stack([one.repeat(16), one.repeat_interleave(16)], 1)  # byte -> (low, high) nibble's values
    rows = both[s["codes"].int()].view(case["n"], -1, 32)
    rows *= torch.exp2(s["scales"].float() - 127.0)[:, :, None]
    rows = rows.view(case["n"], -1)[:, :case["dim"]]
    return s["x"].float() @ rows.t()


def _sequence_of(s, total):
    """(sequence, index among its new tokens) of every new token."""
    at = torch.arange(total, device=DEVICE)
    if s["offsets"] is None:
        return at, torch.zeros_like(at)
    b = torch.searchsorted(s["offsets"][1:].contiguous().long(), at, right=True)
    return b, at - s["offsets"].long()[b]


def _plain_rotate(x, cos, sin):
    """x [T, H, D] f32; the first 2 * cos.shape[1] dimensions rotated, pair (i, i + half)."""
    h = cos.shape[1]
    a, b = x[:, :, :h], x[:, :, h:2 * h]
    c, d = cos[:, None, :], sin[:, None, :]
    return torch.cat([a * c - b * d, b * c + a * d, x[:, :, 2 * h:]], 2)


def _plain_store(codes, scale, x, table, start, end, offsets, page):
    """Writes the new rows x [T, H, D] f32 (positions start..end of their sequences) into the pages."""
    count, heads = table.shape[0], codes.shape[1]
    first = start // page
    grid = first[:, None] + torch.arange(int(x.shape[0]) // page + 2, device=DEVICE)[None, :].clamp(max=table.shape[1])
    touched = (grid * page < end[:, None]) & (grid < table.shape[1]) & (end > start)[:, None]
    b, j = touched.nonzero(as_tuple=True)
    p = grid[b, j]
    pid = table[b, p].long()
    at = p[:, None] * page + torch.arange(page, device=DEVICE)[None, :]
    is_new = (at >= start[b][:, None]) & (at < end[b][:, None])
    is_old = at < start[b][:, None]
    rows = x[(offsets[b][:, None] + at - start[b][:, None]).clamp(0, x.shape[0] - 1)].permute(0, 2, 1, 3)  # [pages, H, P, D]
    rows = torch.where(is_new[:, None, :, None], rows, 0.0)
    m, e = torch.frexp(rows.abs().amax((2, 3)))
    fit = torch.exp2((e - torch.where(m <= 0.875, 9, 8)).clamp(min=-100).float())
    old_scale = scale[pid]
    new_scale = torch.where(is_old.any(1)[:, None], torch.maximum(old_scale, fit), fit)
    old = codes[pid]
    kept = old.float() * (old_scale / new_scale)[:, :, None, None]
    fresh = rows / new_scale[:, :, None, None]
    out = torch.where(is_new[:, None, :, None], fresh, kept).to(torch.float8_e4m3fn).view(torch.uint8)
    out = torch.where((is_new | is_old)[:, None, :, None], out, old.view(torch.uint8))
    codes.view(torch.uint8)[pid] = out
    scale[pid] = new_scale


def _plain_append(s):
    case = s["case"]
    total = s["q"].shape[0]
    b, i = _sequence_of(s, total)
    offsets = torch.arange(case["batch"] + 1, device=DEVICE) if s["offsets"] is None else s["offsets"].long()
    end = s["lengths"].long()
    start = end - (offsets[1:] - offsets[:-1])
    q, k, v = s["q"].float(), s["new_k"].float(), s["new_v"].float()
    if s["cos"] is not None:
        c, d = s["cos"][start[b] + i], s["sin"][start[b] + i]
        q, k = _plain_rotate(q, c, d), _plain_rotate(k, c, d)
    _plain_store(s["k"], s["k_scale"], k, s["table"], start, end, offsets, case["page"])
    _plain_store(s["v"], s["v_scale"], v, s["table"], start, end, offsets, case["page"])
    return q.to(s["q"].dtype), s["k"], s["v"], s["k_scale"], s["v_scale"]


def _plain_gather(codes, scale, table):
    x = codes[table.long()].float() * scale[table.long()][:, :, :, None, None]  # [B, pages, H, P, D]
    return x.permute(0, 2, 1, 3, 4).reshape(x.shape[0], x.shape[2], -1, x.shape[4])


def _plain_softmax(score, seen):
    score = torch.where(seen, score, -torch.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    z = p.sum(-1, keepdim=True)
    return p / z.clamp(min=1e-38), (top + torch.log(z))[..., 0]


def _plain_attend(s):
    case = s["case"]
    B, H, D, G = case["batch"], case["hkv"], case["dim"], case["hq"] // case["hkv"]
    scale = D ** -0.5
    if case["select"]:
        at = s["select"]
        seen = (at >= 0) & (at < s["lengths"].long()[:, None, None])
        at = at.clamp(min=0)
        pid = s["table"].long()[torch.arange(B, device=DEVICE)[:, None, None], at // case["page"]]
        h = torch.arange(H, device=DEVICE)[None, :, None]
        k = s["k"].view(torch.uint8)[pid, h, at % case["page"]].view(torch.float8_e4m3fn).float() * s["k_scale"][pid, h][..., None]
        v = s["v"].view(torch.uint8)[pid, h, at % case["page"]].view(torch.float8_e4m3fn).float() * s["v_scale"][pid, h][..., None]
        score = (s["q"].float().view(B, H, G, D) @ k.transpose(2, 3)) * scale
        p, lse = _plain_softmax(score, seen[:, :, None, :])
        return (p @ v).reshape(B, H * G, D).to(s["q"].dtype), lse.reshape(B, H * G)
    k, v = _plain_gather(s["k"], s["k_scale"], s["table"]), _plain_gather(s["v"], s["v_scale"], s["table"])
    b, i = _sequence_of(s, s["q"].shape[0])
    offsets = torch.arange(B + 1, device=DEVICE) if s["offsets"] is None else s["offsets"].long()
    end = s["lengths"].long()
    N = case["new_max"]
    q = torch.zeros(B, N, H * G, D, device=DEVICE)
    q[b, i] = s["q"].float()
    pos = end[:, None] - (offsets[1:] - offsets[:-1])[:, None] + torch.arange(N, device=DEVICE)[None, :]  # [B, N]
    key = torch.arange(k.shape[2], device=DEVICE)
    seen = (key[None, None, :] <= pos[:, :, None]) & (key[None, None, :] < end[:, None, None])
    if case["window"]:
        seen &= key[None, None, :] > pos[:, :, None] - case["window"]
    q = q.view(B, N, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * N, D)
    score = ((q @ k.transpose(2, 3)) * scale).view(B, H, G, N, -1)
    p, lse = _plain_softmax(score, seen[:, None, None])
    o = (p.view(B, H, G * N, -1) @ v).view(B, H, G, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, H * G, D)
    return o[b, i].to(s["q"].dtype), lse.permute(0, 3, 1, 2).reshape(B, N, H * G)[b, i]


def run(state):
    s = state
    op = s["case"]["op"]
    if not own:
        return {"products": _plain_products, "append": _plain_append, "attend": _plain_attend}[op](s)
    from vectordb_amd.memory import KeyValueMemory
    from vectordb_amd.rows4 import Rows4

    if op == "products":
        return Rows4(s["codes"], s["scales"], s["case"]["dim"]).products(s["x"])
    memory = KeyValueMemory.from_tensors(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if op == "append":
        q = memory.append(s["new_k"], s["new_v"], s["table"], s["lengths"], offsets=s["offsets"], max_new=s["case"]["new_max"],
                          queries=s["q"], cos=s["cos"], sin=s["sin"])
        return q, s["k"], s["v"], s["k_scale"], s["v_scale"]
    return memory.attend(s["q"], s["table"], s["lengths"], offsets=s["offsets"], max_new=s["case"]["new_max"], window=s["case"]["window"],
                         select=s.get("select"), return_lse=True)


def work(case):
    z = SIZE[case["dtype"]]
    if case["op"] == "products":
        groups = -(-case["dim"] // 32)
        return {"bytes": case["n"] * groups * 17 + case["nq"] * case["dim"] * z + 4 * case["n"] * case["nq"], "flops": 2 * case["n"] * case["dim"] * case["nq"]}
    held, new = _lengths(case)
    D, P, hkv, hq = case["dim"], case["page"], case["hkv"], case["hq"]
    if case["op"] == "append":
        total = sum(new)
        old = sum((h - n) % P for h, n in zip(held, new))  # rows that share a page with the first new ones
        pages = sum(-(-h // P) - (h - n) // P for h, n in zip(held, new))
        return {"bytes": total * D * (2 * hq * z + 2 * hkv * z + 2 * hkv) + old * D * hkv * 2 + pages * hkv * 16 + total * case["rot"] * 4,
                "flops": total * case["rot"] * 3 * (hq + hkv) + 4 * total * D * hkv}
    if case["select"]:
        pairs = case["batch"] * case["select"]
        read = pairs
    else:
        w = case["window"] or 1 << 60
        pairs = sum(sum(min(h - n + i + 1, w) for i in range(n)) for h, n in zip(held, new))
        read = sum(min(h, w + n - 1) for h, n in zip(held, new))
    rows = sum(new) * hq
    return {"bytes": 2 * read * hkv * D + rows * (2 * D * z + 4) + (8 * pairs * hkv if case["select"] else 0), "flops": 4 * D * hq * pairs}


# ---- the definitions in 64 bits -----------------------------------------------------------------

def _exact_page(codes, scale, pid, h):
    return codes[pid, h].double() * scale[pid, h].double()


def _exact_products(case, s):
    table = torch.tensor(E2M1, dtype=torch.float64, device=DEVICE)
    out = []
    for lo in range(0, case["n"], 65536):
        byte = s["codes"][lo:lo + 65536].long()
        nib = torch.stack([byte & 15, byte >> 4], 2).flatten(1)[:, :case["dim"]]
        val = table[nib & 7] * (1 - 2 * (nib >> 3)).double()
        exp = s["scales"][lo:lo + 65536].double().repeat_interleave(32, 1)[:, :case["dim"]] - 127
        out.append(s["x"].double() @ (val * 2.0 ** exp).t())
    return torch.cat(out, 1)


def _exact_append(case, s):
    held, new = _lengths(case)
    R = case["rot"]
    k, v = s["new_k"].double(), s["new_v"].double()
    q = s["q"].double()
    at = torch.cat([torch.arange(h - n, h, device=DEVICE) for h, n in zip(held, new)])
    if R:
        c, d = s["cos"].double()[at].unsqueeze(1), s["sin"].double()[at].unsqueeze(1)
        turn = lambda x: torch.cat([x[..., :R // 2] * c - x[..., R // 2:R] * d, x[..., R // 2:R] * c + x[..., :R // 2] * d, x[..., R:]], -1)  # noqa: E731
        q, k = turn(q), turn(k)
    out = []
    for codes, scale, x in ((s["k"], s["k_scale"], k), (s["v"], s["v_scale"], v)):
        val, sc = codes.float(), scale.double().clone()
        done = 0
        for b, (h, n) in enumerate(zip(held, new)):
            start = h - n
            for p in range(start // case["page"], -(-h // case["page"])):
                pid = int(s["table"][b, p])
                lo, hi = max(start, p * case["page"]), min(h, (p + 1) * case["page"])
                rows = x[done + lo - start:done + hi - start].transpose(0, 1)  # [H, rows, D]
                top = rows.abs().amax((1, 2))
                fit = 2.0 ** torch.ceil(torch.log2(top.clamp(min=1e-30) / 448.0)).clamp(min=-100)
                r = lo - p * case["page"]
                if r:
                    use = torch.maximum(sc[pid], fit)
                    val[pid, :, :r] = (val[pid, :, :r] * (sc[pid] / use)[:, None, None].float()).to(torch.float8_e4m3fn).float()
                    fit = use
                sc[pid] = fit
                val[pid, :, r:r + hi - lo] = (rows / fit[:, None, None]).float().to(torch.float8_e4m3fn).float()
            done += n
        out.append((val, sc))
    return q, out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_attend(case, s):
    held, new = _lengths(case)
    H, G, D, P = case["hkv"], case["hq"] // case["hkv"], case["dim"], case["page"]
    outs, lses, done = [], [], 0
    for b, (h, n) in enumerate(zip(held, new)):
        ids = s["table"][b, :-(-h // P)].long()
        o, z = [], []
        pos = torch.arange(h - n, h, device=DEVICE)
        for head in range(H):
            q = s["q"][done:done + n, head * G:(head + 1) * G].double()
            if case["select"]:
                at = s["select"][b, head]
                at = at[at >= 0]
                k = s["k"].view(torch.uint8)[ids[at // P], head, at % P].view(torch.float8_e4m3fn).double() * s["k_scale"][ids[at // P], head].double()[:, None]
                v = s["v"].view(torch.uint8)[ids[at // P], head, at % P].view(torch.float8_e4m3fn).double() * s["v_scale"][ids[at // P], head].double()[:, None]
                hidden = torch.zeros(n, k.shape[0], dtype=torch.bool, device=DEVICE)
            else:
                take = lambda c, sc: (c.view(torch.uint8)[ids, head].view(torch.float8_e4m3fn).double() * sc[ids, head].double()[:, None, None]).reshape(-1, D)[:h]  # noqa: E731
                k, v = take(s["k"], s["k_scale"]), take(s["v"], s["v_scale"])
                key = torch.arange(h, device=DEVICE)
                hidden = key[None, :] > pos[:, None]
                if case["window"]:
                    hidden |= key[None, :] <= pos[:, None] - case["window"]
            score = torch.einsum("ngd,kd->ngk", q, k) / math.sqrt(D)
            score.masked_fill_(hidden[:, None, :], -math.inf)
            o.append(torch.softmax(score, -1) @ v)
            z.append(torch.logsumexp(score, -1))
        outs.append(torch.cat(o, 1))
        lses.append(torch.cat(z, 1))
        done += n
    return torch.cat(outs), torch.cat(lses)


def exact(case, seed):
    s = prepare(case, seed)
    return {"products": _exact_products, "append": _exact_append, "attend": _exact_attend}[case["op"]](case, s)
