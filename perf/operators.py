"""The operators of a paged cache held in 4 bits, case by case: what one pass reads and returns, in elementary torch
operations (`own` false) and through the library's entry points (`own` true).

Four operators make up one step of a serving program over such a cache:

  tables   block tables, slot map and row positions from the requests' lengths         ops.page_tables
  append   per-head norm, rotary positions, K and V quantised into their KV4 cells     ops.rope_neox_kv4_append
  read     cells widened back to F32, by slot                                          ops.kv4_read_f32
  attend   the rows' attention over their requests' pages                              ops.attend_paged_kv4

KV4: groups of 32 values.  m = the value of largest magnitude (the positive one when m and -m both occur),
d = FP16(BF16(m / -8)) with |d| <= 2720, id = F32(1 / d), code = clamp(round_half_even(F32(x id)), -8, 7) + 8, value
(code - 8) d; the codes lie two to a byte in the order of the values, low nibble first.  The planes are
[kv_head][slot][head_dim / 2] bytes and [kv_head][slot][head_dim / 32] FP16 scales.
"""
import math

import numpy as np
import torch

own = False


# ---- the cases ------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step of 64 running requests: one new row each, most of them inside a page they have
        dict(name="tables decode 64", op="tables", n_req=64, old=32768, new=1, page=16, pad=0),
        # a prefill chunk of 65536 rows over 96 requests of very different lengths, in a padded launch
        dict(name="tables prefill 65536", op="tables", n_req=96, old=8192, new=1365, page=16, pad=37),
        # the same decode step's 64 rows into the cache (16 query heads, 2 KV heads of 256, 64 rotary dimensions)
        dict(name="append decode 64", op="append", rows=64, n_q=16, n_kv=2, hd=256, n_rot=64, slots=262144, pad=0),
        # a prefill chunk of 4096 rows at positions far into a long context
        dict(name="append prefill 4096", op="append", rows=4096, n_q=16, n_kv=2, hd=256, n_rot=64, slots=262144, pad=0),
        # an odd number of rows of 128-wide heads rotated over their whole width, the last rows of the launch padding
        dict(name="append 8191 of 128", op="append", rows=8191, n_q=32, n_kv=8, hd=128, n_rot=128, slots=32768, pad=70),
        # a short request's cells read back (a check of a cache, or a move to another tier)
        dict(name="read 333 of 128", op="read", rows=333, n_kv=8, hd=128, slots=4096),
        # a long request's cells read back by their slots
        dict(name="read 65536 of 256", op="read", rows=65536, n_kv=2, hd=256, slots=262144),
        # a few short chats: latency counts
        dict(name="attend 8 short", op="attend", n_req=8, cells=300, rows=1, n_q=16, n_kv=2, hd=256, page=16, gate=False),
        # one request at the full depth, one new row
        dict(name="attend 196608 deep", op="attend", n_req=1, cells=196608, rows=1, n_q=16, n_kv=2, hd=256, page=64, gate=True),
        # a batch of 64 requests of ragged lengths, one row each
        dict(name="attend 64 ragged", op="attend", n_req=64, cells=8192, rows=1, n_q=16, n_kv=2, hd=256, page=16, gate=True),
        # 13 requests that each verify one to five drafted rows, 12 query heads on one KV head
        dict(name="attend 13 drafts", op="attend", n_req=13, cells=16384, rows=5, n_q=12, n_kv=1, hd=256, page=32, gate=True),
        # 128-wide heads in groups of four, larger pages
        dict(name="attend 40 of 128", op="attend", n_req=40, cells=5000, rows=1, n_q=32, n_kv=8, hd=128, page=128, gate=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("tables", "append", "read", "attend", "attend"))
    if op == "tables":
        return dict(op=op, n_req=_log_int(rng, 1, 1000), old=_log_int(rng, 1, 32768), new=_log_int(rng, 1, 64),
                    page=rng.choice((16, 32, 64, 128, 256)), pad=rng.randrange(0, 100))
    hd = rng.choice((64, 128, 256))
    n_kv = rng.choice((1, 2, 4, 8)) if hd < 256 else rng.choice((1, 2))
    if op == "append":
        return dict(op=op, rows=_log_int(rng, 1, 4000), n_q=n_kv * rng.choice((1, 2, 4, 8)), n_kv=n_kv, hd=hd,
                    n_rot=rng.choice((0, 64) if hd == 64 else (64, 128)), slots=_log_int(rng, 5000, 100000), pad=rng.randrange(0, 20))
    if op == "read":
        return dict(op=op, rows=_log_int(rng, 1, 30000), n_kv=n_kv, hd=hd, slots=_log_int(rng, 30000, 200000))
    n_req = _log_int(rng, 1, 64)
    return dict(op=op, n_req=n_req, cells=_log_int(rng, 1, max(2, 300000 // n_req // n_kv)), rows=rng.choice((1, 1, 1, 2, 3, 5)),
                n_q=n_kv * rng.choice((1, 3, 4, 6, 8, 12)), n_kv=n_kv, hd=hd, page=rng.choice((16, 32, 64, 128, 256)),
                gate=rng.random() < 0.5)


# ---- what a case fixes apart from the values: ragged lengths, spread evenly by multiples of the golden ratio -----------

def _spread(n, top, k):
    """n whole numbers in [1, top], the largest of them top."""
    v = [1 + int((top - 1) * (((i + 1) * k * 0.6180339887498949) % 1.0)) for i in range(n)]
    v[n // 2] = top
    return v


def _table_lengths(c):
    old = [0 if i % 7 == 3 else v for i, v in enumerate(_spread(c["n_req"], c["old"], 1))]
    new = [1] * c["n_req"] if c["new"] == 1 else [0 if i % 11 == 5 else v for i, v in enumerate(_spread(c["n_req"], c["new"], 3))]
    return old, new


def _attend_lengths(c):
    rows = [1] * c["n_req"] if c["rows"] == 1 else _spread(c["n_req"], c["rows"], 3)
    return [max(n, m) for n, m in zip(_spread(c["n_req"], c["cells"], 1), rows)], rows


def _pages(n, page):
    return (n + page - 1) // page


def _theta(n_rot):
    return float(np.float32(1e7 ** (-2.0 / n_rot))) if n_rot else 1.0


# ---- inputs --------------------------------------------------------------------------------------------------------------

def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32).to(dev)


def _cells(g, n_kv, slots, hd, dev):
    """Codes and scales as a quantiser leaves them: nearly Gaussian codes, scales of either sign in BF16 steps."""
    code = (torch.randn((n_kv, slots, hd), generator=g, device=dev) * 2.9).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
    codes = code[..., 0::2] | (code[..., 1::2] << 4)
    d = (torch.randn((n_kv, slots, hd // 32), generator=g, device=dev) * 0.2).exp_() * 0.3
    d = torch.where(torch.rand(d.shape, generator=g, device=dev) < 0.5, -d, d)
    return codes.contiguous(), d.to(torch.bfloat16).to(torch.float16).view(torch.int16)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(dev)
    g.manual_seed(seed)
    c = dict(case)
    if c["op"] == "tables":
        old, new = _table_lengths(c)
        max_pages = max(_pages(o + n, c["page"]) for o, n in zip(old, new)) + 3
        held = [_pages(o, c["page"]) for o in old]
        n_pages = sum(_pages(o + n, c["page"]) for o, n in zip(old, new)) + 50
        perm = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
        at = torch.cumsum(torch.tensor(held), 0) - torch.tensor(held)
        j = torch.arange(max_pages)[None, :]
        has = j < torch.tensor(held)[:, None]
        index = torch.where(has, at[:, None] + j, 0).to(dev)
        table = torch.where(has.to(dev), perm[index], -1).to(torch.int32).contiguous()
        return dict(c=c, table=table, n_old=_i32(old, dev), n_new=_i32(new, dev), free=perm[sum(held):].contiguous(),
                    head=_i32([5], dev), rows=sum(new) + c["pad"], n_pages=n_pages,
                    grown=sum(_pages(o + n, c["page"]) for o, n in zip(old, new)) - sum(held))
    if c["op"] == "append":
        rows, hd, total = c["rows"], c["hd"], c["rows"] + c["pad"]
        slots = torch.randperm(c["slots"], generator=g, device=dev)[:total].to(torch.int32)
        slots[rows:] = -1
        first = int(torch.randint(0, 258048, (1,), generator=g, device=dev))
        pos = (torch.arange(total, device=dev) + first).to(torch.int32)
        weight = lambda: 1.0 + 0.1 * torch.randn(hd, generator=g, device=dev)  # noqa: E731
        codes = lambda: torch.zeros((c["n_kv"], c["slots"], hd // 2), dtype=torch.uint8, device=dev)  # noqa: E731
        scales = lambda: torch.zeros((c["n_kv"], c["slots"], hd // 32), dtype=torch.int16, device=dev)  # noqa: E731
        normal = lambda n: torch.randn((total, n, hd), generator=g, device=dev)  # noqa: E731
        return dict(c=c, q=normal(c["n_q"]), k=normal(c["n_kv"]), v=normal(c["n_kv"]), pos=pos, slots=slots, wq=weight(),
                    wk=weight(), k_cache=codes(), v_cache=codes(), k_scale=scales(), v_scale=scales(),
                    q_out=torch.zeros((total, c["n_q"], hd), device=dev), live=slots[:rows].contiguous())
    if c["op"] == "read":
        codes, scale = _cells(g, c["n_kv"], c["slots"], c["hd"], dev)
        return dict(c=c, codes=codes, scale=scale, cells=torch.randperm(c["slots"], generator=g, device=dev)[: c["rows"]].to(torch.int32))
    lens, rows = _attend_lengths(c)
    page, hd = c["page"], c["hd"]
    need = [_pages(n, page) for n in lens]
    n_pages = sum(need) + 7
    slots = n_pages * page
    kc, ks = _cells(g, c["n_kv"], slots, hd, dev)
    vc, vs = _cells(g, c["n_kv"], slots, hd, dev)
    max_pages = max(need)
    perm = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    at = torch.cumsum(torch.tensor(need), 0) - torch.tensor(need)
    j = torch.arange(max_pages)[None, :]
    has = j < torch.tensor(need)[:, None]
    table = torch.where(has.to(dev), perm[torch.where(has, at[:, None] + j, 0).to(dev)], -1).to(torch.int32).contiguous()
    # the cells behind a request's last one were never written: their scales are NaN
    last = torch.tensor([n - 1 for n in lens])
    tail = torch.arange(page)[None, :] > (last % page)[:, None]
    end = perm[(at + last // page).to(dev)].long()[:, None] * page + torch.arange(page, device=dev)[None, :]
    for s in (ks, vs):
        s[:, end[tail.to(dev)]] = 0x7E00
    total = sum(rows)
    q = torch.randn((total, c["n_q"], hd), generator=g, device=dev)
    starts = [0]
    for m in rows:
        starts.append(starts[-1] + m)
    return dict(c=c, q=q, gate=torch.randn(q.shape, generator=g, device=dev) if c["gate"] else None, k_cache=kc, v_cache=vc,
                k_scale=ks, v_scale=vs, table=table, n_cells=_i32(lens, dev), row_start=_i32(starts, dev),
                max_rows=max(rows), max_cells=max(lens), out=torch.zeros_like(q))


# ---- one pass ------------------------------------------------------------------------------------------------------------

def run(state):
    c = state["c"]
    if own:
        from fnfl_v100_b200 import ops
        if c["op"] == "tables":
            t = ops.page_tables(state["table"], state["n_old"], state["n_new"], state["free"], page_size=c["page"],
                                n_pages=state["n_pages"], rows=state["rows"], free_head=state["head"])
            return dict(table=state["table"], slots=t.slots, pos=t.pos, row_start=t.row_start, n_cells=t.n_cells, head=t.free_head)
        if c["op"] == "append":
            ops.rope_neox_kv4_append(state["q"], state["k"], state["v"], state["pos"], n_rot=c["n_rot"], theta_scale=_theta(c["n_rot"]),
                                     k_cache=state["k_cache"], v_cache=state["v_cache"], k_scale=state["k_scale"],
                                     v_scale=state["v_scale"], slots=state["slots"], q_norm_w=state["wq"], k_norm_w=state["wk"],
                                     q_out=state["q_out"])
            # the cells as the values they stand for
            return dict(q=state["q_out"], k=ops.kv4_read_f32(state["k_cache"], state["k_scale"], cells=state["live"]),
                        v=ops.kv4_read_f32(state["v_cache"], state["v_scale"], cells=state["live"]))
        if c["op"] == "read":
            return ops.kv4_read_f32(state["codes"], state["scale"], cells=state["cells"])
        return ops.attend_paged_kv4(state["q"], state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"], state["table"],
                                    state["n_cells"], page_size=c["page"], row_start=state["row_start"], max_rows=state["max_rows"],
                                    gate=state["gate"], out=state["out"])
    if c["op"] == "tables":
        return _plain_tables(state)
    if c["op"] == "append":
        return _plain_append(state)
    if c["op"] == "read":
        slots = state["cells"].long()
        return _widen(state["codes"][:, slots], state["scale"][:, slots]).transpose(0, 1).contiguous()
    return _plain_attend(state)


def _plain_tables(s):
    page, table, rows = s["c"]["page"], s["table"], s["rows"]
    n_req = table.shape[0]
    old, new = s["n_old"].long(), s["n_new"].long()
    held = (old + page - 1) // page
    grow = (old + new + page - 1) // page - held
    row_end, page_end = torch.cumsum(new, 0), torch.cumsum(grow, 0)
    # new pages: the i-th goes to the request whose share of the free list holds i
    i = torch.arange(s["grown"], device=table.device)
    r = torch.searchsorted(page_end, i, right=True)
    table[r, held[r] + i - (page_end - grow)[r]] = s["free"][s["head"].long() + i]
    # rows
    i = torch.arange(rows, device=table.device)
    r = torch.searchsorted(row_end, i, right=True)
    live = r < n_req
    r = r.clamp(max=n_req - 1)
    pos = old[r] + i - (row_end - new)[r]
    slot = table[r, (pos // page).clamp(max=table.shape[1] - 1)].long() * page + pos % page
    start = torch.cat((torch.zeros_like(row_end[:1]), row_end))
    int32 = torch.int32
    return dict(table=table, slots=torch.where(live, slot, -1).to(int32), pos=torch.where(live, pos, -1).to(int32),
                row_start=start.to(int32), n_cells=(old + new).to(int32), head=(s["head"].long() + page_end[-1:]).to(int32))


def _widen(codes, scale):
    """(code - 8) d in F32: codes [..., hd / 2] and scales [..., hd / 32] to values [..., hd]."""
    v = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8.0
    return (v.unflatten(-1, (-1, 32)) * scale.view(torch.float16).float().unsqueeze(-1)).flatten(-2)


def _quantised(x):
    """The values the cells of x stand for."""
    g = x.unflatten(-1, (-1, 32))
    top, low = g.amax(-1, keepdim=True), g.amin(-1, keepdim=True)
    d = (torch.where(top >= -low, top, low) / -8.0).to(torch.bfloat16).float().clamp(-2720.0, 2720.0).to(torch.float16).float()
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    return ((g * inv).round().clamp(-8, 7) * d).flatten(-2)


def _plain_norm(x, w, eps=1e-6):
    mean = ((x * x).double().sum(-1, keepdim=True) / x.shape[-1]).float()
    return x * (1.0 / torch.sqrt(mean + eps)) * w


def _plain_rope(x, pos, n_rot):
    if not n_rot:
        return x
    half = n_rot // 2
    # the angle is defined as an F32 product chain, position times theta once for each pair before it
    steps = [pos.float()]
    for _ in range(half - 1):
        steps.append(steps[-1] * _theta(n_rot))
    angle = torch.stack(steps, -1).double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., :half], x[..., half:n_rot]
    return torch.cat((a * cos - b * sin, a * sin + b * cos, x[..., n_rot:]), -1)


def _plain_append(s):
    c, live = s["c"], (s["slots"] >= 0)[:, None, None]
    q = _plain_rope(_plain_norm(s["q"], s["wq"]), s["pos"], c["n_rot"])
    k = _plain_rope(_plain_norm(s["k"], s["wk"]), s["pos"], c["n_rot"])
    return dict(q=torch.where(live, q, torch.zeros_like(q)), k=_quantised(k[: c["rows"]]), v=_quantised(s["v"][: c["rows"]]))


def _plain_attend(s):
    c, q = s["c"], s["q"]
    page, n_kv, hd = c["page"], c["n_kv"], c["hd"]
    n_req, top, dev = c["n_req"], s["max_cells"], q.device
    cell = torch.arange(top, device=dev)
    held = cell[None, :] < s["n_cells"][:, None]                                            # [req][cell]
    slot = torch.where(held, s["table"].long()[:, cell // page] * page + cell % page, 0)
    widen = lambda codes, scale: torch.where(held[None, :, :, None], _widen(codes[:, slot], scale[:, slot]), 0.0)  # noqa: E731
    # rows of a request side by side: [req][kv head][row, head of the group][hd]
    m = (s["row_start"][1:] - s["row_start"][:-1]).long()
    j = torch.arange(s["max_rows"], device=dev)
    row = (s["row_start"][:-1].long()[:, None] + j[None, :]).clamp(max=q.shape[0] - 1)
    group = c["n_q"] // n_kv
    x = q[row].view(n_req, -1, n_kv, group, hd).permute(2, 0, 1, 3, 4).reshape(n_kv, n_req, -1, hd)
    score = torch.matmul(x, widen(s["k_cache"], s["k_scale"]).transpose(-1, -2)) * hd ** -0.5
    sees = cell[None, None, :] <= (s["n_cells"].long() - m)[:, None, None] + j[None, :, None]  # [req][row][cell]
    sees = sees.repeat_interleave(group, 1)[None]
    score = torch.where(sees, score, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = torch.matmul(p, widen(s["v_cache"], s["v_scale"])) / p.sum(-1, keepdim=True)
    out = out.view(n_kv, n_req, -1, group, hd).permute(1, 2, 0, 3, 4).reshape(n_req, -1, c["n_q"], hd)
    out = out[j[None, :] < m[:, None]]
    return out * torch.sigmoid(s["gate"]) if s["gate"] is not None else out


# ---- the work of a pass ----------------------------------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "tables":
        old, new = _table_lengths(c)
        grow = sum(_pages(o + n, c["page"]) - _pages(o, c["page"]) for o, n in zip(old, new))
        # lengths in and out, the new pages out of the list and into the table, a table entry, slot and position a row
        rows = sum(new)
        return {"bytes": 4 * (4 * c["n_req"] + 1 + 2 * grow + 2 * (rows + c["pad"]) + sum(_pages(n, c["page"]) for n in new)), "flops": 0}
    hd, n_kv = c["hd"], c["n_kv"]
    cell = n_kv * (hd // 2 + hd // 16)  # one plane's codes and scales of a slot
    if c["op"] == "append":
        row = (2 * c["n_q"] + 2 * n_kv) * hd * 4 + 2 * cell + 8
        return {"bytes": c["rows"] * (row + 2 * cell + 2 * n_kv * hd * 4), "flops": c["rows"] * (c["n_q"] + 2 * n_kv) * hd * 10}
    if c["op"] == "read":
        return {"bytes": c["rows"] * (cell + n_kv * hd * 4 + 4), "flops": c["rows"] * n_kv * hd}
    lens, rows = _attend_lengths(c)
    vectors = 3 if c["gate"] else 2
    return {"bytes": sum(lens) * 2 * cell + sum(rows) * c["n_q"] * hd * 4 * vectors + 4 * sum(_pages(n, c["page"]) for n in lens),
            "flops": sum(4 * c["n_q"] * hd * (n - m + i + 1) for n, m in zip(lens, rows) for i in range(m))}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------

def exact(case, seed):
    c = case
    if c["op"] == "tables":
        return None  # whole numbers
    s = prepare(case, seed)
    if c["op"] == "read":
        return _decoded(s["codes"], s["scale"])[:, s["cells"].long()].permute(1, 0, 2)
    if c["op"] == "append":
        # the cells are codes: rounded to a format, they have no value of their own in 64 bits
        live = (s["slots"] >= 0).double()[:, None, None]
        x = s["q"].double()
        x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * s["wq"].double()
        if c["n_rot"]:
            half = c["n_rot"] // 2
            angle = np.empty((s["pos"].numel(), half), np.float32)  # the chain's own F32 roundings belong to the definition
            angle[:, 0] = s["pos"].cpu().numpy().astype(np.float32)
            for i in range(1, half):
                angle[:, i] = angle[:, i - 1] * np.float32(_theta(c["n_rot"]))
            turn = torch.polar(torch.ones((), dtype=torch.float64), torch.from_numpy(angle.astype(np.float64))).to(x.device)
            pair = torch.complex(x[..., :half], x[..., half: c["n_rot"]]) * turn[:, None]
            x = torch.cat((pair.real, pair.imag, x[..., c["n_rot"]:]), -1)
        return dict(q=x * live, k=None, v=None)
    page, group = c["page"], c["n_q"] // c["n_kv"]
    lens, rows = _attend_lengths(c)
    out = torch.empty_like(s["q"], dtype=torch.float64)
    at = 0
    for r, (n, m) in enumerate(zip(lens, rows)):
        slot = (s["table"][r, : _pages(n, page)].long()[:, None] * page + torch.arange(page, device=s["q"].device)).reshape(-1)[:n]
        for h in range(c["n_kv"]):
            k, v = (_decoded(s[x + "_cache"][h, slot], s[x + "_scale"][h, slot]) for x in "kv")
            for i in range(m):
                upto = n - m + i + 1
                w = torch.softmax((s["q"][at + i, h * group: (h + 1) * group].double() @ k[:upto].T) / math.sqrt(c["hd"]), -1)
                out[at + i, h * group: (h + 1) * group] = w @ v[:upto]
        at += m
    return out / (1.0 + torch.exp(-s["gate"].double())) if c["gate"] else out


def _decoded(codes, scale):
    v = torch.empty(codes.shape[:-1] + (codes.shape[-1] * 2,), dtype=torch.float64, device=codes.device)
    v[..., 0::2] = (codes % 16).double() - 8
    v[..., 1::2] = torch.div(codes, 16, rounding_mode="floor").double() - 8
    return v * scale.view(torch.float16).double().repeat_interleave(32, -1)
