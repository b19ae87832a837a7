"""The operators of the e4m3 cache (pool format TGE_KV_E4M3), as measurable cases.

The cache holds K and V as OCP e4m3 codes in pages of 16 tokens. The 16
tokens of one KV head are a block; its K codes share one power of two 2^e and
its V codes another (bf16), so a stored value is code * 2^e, -15 <= e <= 7.

  append  a step's new rows of K and V go into their pages. Per block,
          e = the smallest exponent with max|x| <= 448 * 2^e over the block's
          new rows; where the block already holds rows, never below their e.
          x is stored as the code nearest x * 2^-e (ties to even); rows that
          were there before are re-encoded when e grew; the slots behind the
          last new row are cleared. With `rope` the step before the store is
          part of it: biases are added to q, k and v, then q and k are rotated
          (halves of a head against each other), q into a buffer of its own.
  attend  softmax(q K^T / sqrt(head_dim)) V over a session's pages; new token
          i of a session sees the positions 0 .. ctx + i. Sessions with a few
          new tokens (decode, drafted tokens to verify), prompt chunks, or
          both kinds in one step.

Rows of q, k, v and out are bf16 or f16; `fused` rows are slices of one
projection's output (a row stride larger than the row).
"""
import math
import os
import sys

import torch

own = False

# name: query heads, KV heads, head dim
SHAPES = {
    "0.5b": (14, 2, 64),
    "1.5b": (12, 2, 128),
    "7b": (28, 4, 128),
    "wide": (16, 8, 256),
    "h96": (16, 4, 96),  # a head size between the block widths
}
OUTLIER_GAIN = 8.0  # 1 % of the K channels carry outliers


def _case(name, op, shape, rows, **more):
    c = {"name": name, "op": op, "shape": shape, "rows": rows, "contexts": "", "n_new": 1, "start": 0, "count": 0,
         "rope": False, "fused": False}
    c.update(more)
    return c


def _text(values):
    return ",".join(str(int(v)) for v in values)


def _log_spread(n, lo, hi, turn):
    """n contexts spread over [lo, hi] in equal steps of their logarithm, in a mixed order."""
    v = [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]
    return [v[i * turn % n] for i in range(n)]


def listed():
    serve = _log_spread(64, 1024, 32768, 27)
    return [
        # one user chatting: one new token's rows, the launch's latency
        _case("append-chat", "append", "7b", "bf16", contexts="1056", rope=True, fused=True),
        # 64 sessions of ragged contexts, four drafted tokens each: pages written in part
        _case("append-serve", "append", "7b", "bf16", contexts=_text(serve), n_new=4, rope=True, fused=True),
        # a prompt chunk of the 256-dim shape behind a cached prefix that ends inside a page
        _case("append-wide-chunk", "append", "wide", "f16", start=777, count=2048, rope=True),
        # a long prefix restored into the cache, without rotation
        _case("append-prefix", "append", "7b", "bf16", count=20000),
        # one user chatting with a small model
        _case("attend-chat", "attend", "0.5b", "f16", contexts="1056"),
        # a handful of sessions of ragged lengths
        _case("attend-four", "attend", "1.5b", "bf16", contexts="527,2063,4111,8207"),
        # serving: 64 sessions of 1k to 32k tokens, four drafted tokens each
        _case("attend-serve", "attend", "7b", "bf16", contexts=_text(serve), n_new=4, fused=True),
        # 256-dim heads, 32 sessions, one new token each
        _case("attend-serve-wide", "attend", "wide", "bf16", contexts=_text(_log_spread(32, 1024, 32768, 13))),
        # a whole short prompt of ragged length, a head size between the block widths
        _case("attend-prompt-h96", "attend", "h96", "f16", count=777),
        # a prompt's last chunk of 512 tokens
        _case("attend-chunk", "attend", "7b", "bf16", start=1536, count=512, fused=True),
        # a long message late in a conversation
        _case("attend-turn", "attend", "7b", "bf16", start=14003, count=1333, fused=True),
        # 32 verifying sessions beside a prompt chunk in one step
        _case("attend-mixed", "attend", "7b", "bf16", contexts=_text(serve[:32]), n_new=4, start=1536, count=512,
              fused=True),
    ]


def _span(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_MOST = {}


def _most(op):
    if op not in _MOST:
        w = [work(c) for c in listed() if c["op"] == op]
        _MOST[op] = (max(x["bytes"] for x in w), max(x["flops"] for x in w))
    return _MOST[op]


def draw(rng):
    while True:
        op = rng.choice(["append", "attend", "attend"])
        kind = rng.choice(["decode", "decode", "prompt", "mixed"])
        shape = rng.choice(sorted(SHAPES))
        c = _case("", op, shape, rng.choice(["bf16", "bf16", "f16"]))
        del c["name"]
        qh, kvh, _ = SHAPES[shape]
        if kind != "prompt":
            hi = rng.choice([1024, 8192, 32768])
            c["contexts"] = _text(_span(rng, 1, hi) - 1 for _ in range(_span(rng, 1, 64)))
            c["n_new"] = rng.choice([1, 1, 2, 3, 4, 6])
        if kind != "decode":
            c["start"] = rng.choice([0, _span(rng, 1, 14003)])
            c["count"] = _span(rng, 7, 20000 if op == "append" else 2048)
        c["rope"] = op == "append" and rng.random() < 0.6
        c["fused"] = rng.random() < 0.5
        w = work(c)
        if w["bytes"] <= _most(op)[0] and w["flops"] <= _most(op)[1]:
            return c


def _sessions(case):
    """(cached tokens, new tokens, first row of the step) of each session."""
    got, row = [], 0
    for ctx in ([int(x) for x in case["contexts"].split(",")] if case["contexts"] else []):
        got.append((ctx, case["n_new"], row))
        row += case["n_new"]
    if case["count"]:
        got.append((case["start"], case["count"], row))
    return got


def work(case):
    """append: the new rows in, their codes out, two bytes of scale for each
    block's part (read where the block was begun before); with rope q in and out and the
    tables' rows. attend: q in, out, every cached code and scale that a
    session's queries see, once, and the page ids; flops of the two products."""
    qh, kvh, hd = SHAPES[case["shape"]]
    nbytes = flops = 0
    for ctx, n, _ in _sessions(case):
        pages = -(-(ctx + n) // 16)
        if case["op"] == "append":
            touched = pages - ctx // 16
            nbytes += n * 2 * kvh * hd * (2 + 1) + (touched + (ctx % 16 > 0)) * kvh * 4 + touched * 4
            if case["rope"]:
                nbytes += n * (2 * 2 * qh * hd + hd * 4)
                flops += 3 * n * (qh + kvh) * hd
        else:
            nbytes += 2 * 2 * n * qh * hd + (ctx + n) * 2 * kvh * hd + pages * (4 * kvh + 4)
            flops += 4 * qh * hd * (n * ctx + n * (n + 1) // 2)
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _block_width(hd):
    return 64 if hd <= 64 else 128 if hd <= 128 else 256


def _order(width):
    """Places of (token, dim) in a block of 2 * 16 * width codes: [2][16][width]
    (K, V). A part is a sequence of KiB of 64 lanes x 16 bytes."""
    t = torch.arange(16, device="cuda")[:, None]
    d = torch.arange(width, device="cuda")[None, :]

    def place(lane, j):
        return (j // 16 * 64 + lane) * 16 + j % 16

    k = place((d // 16 % 4) * 16 + t, d // 64 * 16 + d % 16)
    v = place(t // 4 * 16 + d % 16, d // 16 % 2 * (width // 8) + d // 32 * 4 + t % 4)
    return torch.stack([k, v + 16 * width])


def _exponent(most):
    """The smallest e with most <= 448 * 2^e, within -15 .. 7 (448 = 0.875 * 2^9)."""
    m, x = torch.frexp(most)
    e = torch.where(m <= 0.875, x - 9, x - 8)
    return torch.where(most > 0, e, torch.full_like(e, -15)).clamp(-15, 7)


def _power(e):
    return torch.ldexp(torch.ones((), device="cuda"), e)


def _codes(x, e):
    y = torch.ldexp(x, -e).clamp(-448.0, 448.0)
    return torch.where(y == y, y, torch.zeros_like(y)).to(torch.float8_e4m3fn)


def _inputs(case, seed):
    """A layer's pages as they are before the call, the block tables and the step's rows."""
    qh, kvh, hd = SHAPES[case["shape"]]
    width = _block_width(hd)
    sessions = _sessions(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 29)
    counts = [-(-(ctx + n) // 16) for ctx, n, _ in sessions]
    pages = sum(counts) + sum(counts) // 16 + 8  # a pool with room left
    ids = torch.randperm(pages, generator=g, device="cuda")[: sum(counts)]
    # rows that each page of the tables holds before the call
    cached = torch.cat([torch.arange(c, device="cuda") * -16 + ctx + (n if case["op"] == "attend" else 0)
                        for (ctx, n, _), c in zip(sessions, counts)]).clamp(0, 16)
    order = _order(width)
    blocks = torch.zeros((pages, kvh, 2 * 16 * width), dtype=torch.uint8, device="cuda")
    scales = torch.zeros((pages, kvh, 2), dtype=torch.bfloat16, device="cuda")
    loud = torch.ones((kvh, 1, hd), device="cuda")
    loud.view(-1)[torch.randperm(kvh * hd, generator=g, device="cuda")[: math.ceil(0.01 * kvh * hd)]] = OUTLIER_GAIN
    live = (torch.arange(16, device="cuda") < cached[:, None])[:, None, :, None]
    for part in range(2):
        x = torch.randn((len(ids), kvh, 16, hd), generator=g, device="cuda") * live
        if part == 0:
            x = x * loud
        e = _exponent(x.abs().amax((-1, -2)))
        c = torch.zeros((len(ids), kvh, 16, width), dtype=torch.uint8, device="cuda")
        c[..., :hd] = _codes(x, e[..., None, None]).view(torch.uint8)
        flat = torch.empty((len(ids), kvh, 16 * width), dtype=torch.uint8, device="cuda")
        flat[..., order[part].reshape(-1) - part * 16 * width] = c.reshape(len(ids), kvh, 16 * width)
        blocks[ids, :, part * 16 * width: (part + 1) * 16 * width] = flat
        scales[ids, :, part] = _power(e).bfloat16()
        del x, c, flat
    rows = sum(n for _, n, _ in sessions)
    kind = torch.bfloat16 if case["rows"] == "bf16" else torch.float16
    x = torch.randn((rows, (qh + 2 * kvh) * hd), generator=g, device="cuda")
    x[:, qh * hd: (qh + kvh) * hd] *= loud.reshape(-1)
    x = x.to(kind)
    q, k, v = x.split([qh * hd, kvh * hd, kvh * hd], 1)
    if not case["fused"]:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    got = {"ids": ids, "blocks": blocks, "scales": scales, "order": order, "q": q, "k": k, "v": v, "pages": pages,
           "tables": torch.split(ids, counts), "keep": x}
    if case["rope"]:
        for name, n in (("q_bias", qh * hd), ("k_bias", kvh * hd), ("v_bias", kvh * hd)):
            got[name] = torch.randn((n,), generator=g, device="cuda")
        pos = torch.arange(max(ctx + n for ctx, n, _ in sessions), device="cuda", dtype=torch.float64)
        freq = 1e6 ** (-2.0 * torch.arange(hd // 2, device="cuda", dtype=torch.float64) / hd)
        got["cos"] = torch.cos(pos[:, None] * freq).float().contiguous()
        got["sin"] = torch.sin(pos[:, None] * freq).float().contiguous()
    return got


class _Memory:
    """A library allocation for torch to look at; a tensor over it keeps the owner."""

    def __init__(self, ptr, shape, kind, owner):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": shape, "typestr": kind, "data": (ptr, False), "version": 3}


def prepare(case, seed):
    qh, kvh, hd = SHAPES[case["shape"]]
    x = _inputs(case, seed)
    sessions = _sessions(case)
    rows = x["q"].shape[0]
    state = dict(x, case=case)
    state["out"] = torch.empty((rows, qh * hd), dtype=x["q"].dtype, device="cuda")
    if own:
        # the library's pool holds the pages; the plan serves every layer of a step
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "aegean-tge_amd"))
        import tge_kv as tk
        pool = tk.KvPool(1, x["pages"], kvh, hd, tk.KV_E4M3)
        view = pool.layer(0)
        state["blocks"] = torch.as_tensor(_Memory(view.k, tuple(x["blocks"].shape), "|u1", pool), device="cuda")
        state["scales"] = torch.as_tensor(_Memory(view.k_scales, tuple(x["scales"].shape), "<i2", pool),
                                          device="cuda").view(torch.bfloat16)
        state["blocks"].copy_(x["blocks"])
        state["scales"].copy_(x["scales"])
        batch = tk.Batch().plan(pool, [tk.Session(ctx, n, t.tolist()) for (ctx, n, _), t in zip(sessions, x["tables"])], qh)
        kind = tk.ROWS_BF16 if case["rows"] == "bf16" else tk.ROWS_F16
        q, k, v, out = x["q"], x["k"], x["v"], state["out"]
        if case["op"] == "append":
            more = {}
            if case["rope"]:
                more = dict(q=q.data_ptr(), q_stride=q.stride(0), q_out=out.data_ptr(), q_out_stride=out.stride(0),
                            q_bias=x["q_bias"].data_ptr(), k_bias=x["k_bias"].data_ptr(), v_bias=x["v_bias"].data_ptr(),
                            rope_cos=x["cos"].data_ptr(), rope_sin=x["sin"].data_ptr(), rope_positions=x["cos"].shape[0])
            args = tk.append_rows_args(kind, k.data_ptr(), v.data_ptr(), k_stride=k.stride(0), v_stride=v.stride(0), **more)
        else:
            args = tk.attention_rows_args(kind, q.data_ptr(), out.data_ptr(), q_stride=q.stride(0), out_stride=out.stride(0))
        state.update(pool=pool, batch=batch, args=args)
    elif case["op"] == "append":
        # the plan: each new row's page and slot, each touched page's first new slot
        pos = torch.cat([torch.arange(ctx, ctx + n, device="cuda") for ctx, n, _ in sessions])
        page = torch.cat([t[torch.arange(ctx, ctx + n, device="cuda") // 16]
                          for (ctx, n, _), t in zip(sessions, x["tables"])])
        touched = torch.cat([t[ctx // 16:] for (ctx, n, _), t in zip(sessions, x["tables"])])
        begun = torch.cat([((ctx - torch.arange(ctx // 16, ctx // 16 + len(t[ctx // 16:]), device="cuda") * 16).clamp(0, 16))
                           for (ctx, n, _), t in zip(sessions, x["tables"])])
        place = torch.empty((x["pages"],), dtype=torch.int64, device="cuda")
        place[touched] = torch.arange(len(touched), device="cuda")
        state.update(pos=pos, tile=place[page], touched=touched, begun=begun)
    return state


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _rotated(x, bias, cos, sin, hd):
    """x + bias, then the rotation with one rounding of h*s (h*c) and one of the sum, as a fused multiply-add has them."""
    y = (x.float() + bias).view(x.shape[0], -1, hd)
    lo, hi = y[..., : hd // 2], y[..., hd // 2:]
    a = (lo.double() * cos.double() - (hi * sin).double()).float()
    b = (lo.double() * sin.double() + (hi * cos).double()).float()
    return torch.cat([a, b], -1).reshape(x.shape[0], -1)


def _append(state):
    case = state["case"]
    qh, kvh, hd = SHAPES[case["shape"]]
    width = _block_width(hd)
    k, v = state["k"].float(), state["v"].float()
    got = {}
    if case["rope"]:
        cos, sin = state["cos"][state["pos"]][:, None], state["sin"][state["pos"]][:, None]
        state["out"].copy_(_rotated(state["q"], state["q_bias"], cos, sin, hd))
        got["q"] = state["out"]
        k = _rotated(state["k"], state["k_bias"], cos, sin, hd)
        v = v + state["v_bias"]
    touched, begun = state["touched"], state["begun"]
    old = torch.arange(16, device="cuda") < begun[:, None]
    mine = state["blocks"][touched]
    for part, rows in ((0, k), (1, v)):
        x = torch.zeros((len(touched), 16, kvh, width), device="cuda")
        x[state["tile"], state["pos"] % 16, :, :hd] = rows.view(-1, kvh, hd)
        x = x.transpose(1, 2)
        e = _exponent(torch.where(x == x, x.abs(), torch.zeros_like(x)).amax((-1, -2)))
        had = torch.frexp(state["scales"][touched, :, part].float())[1] - 1
        e = torch.where(begun[:, None] > 0, torch.maximum(e, had), e)
        at = state["order"][part].reshape(-1)
        was = mine[..., at].view(torch.float8_e4m3fn).float().view(len(touched), kvh, 16, width)
        was = _codes(torch.ldexp(was, had[..., None, None]), e[..., None, None]).view(torch.uint8)
        now = _codes(x, e[..., None, None]).view(torch.uint8)
        mine[..., at] = torch.where(old[:, None, :, None], was, now).reshape(len(touched), kvh, 16 * width)
        state["scales"][touched, :, part] = _power(e).bfloat16()
    state["blocks"][touched] = mine
    return got


def _values(state, table, part, hd):
    """The rows [KV head][token][dim] that a session's pages hold."""
    width = _block_width(hd)
    c = state["blocks"][table][..., state["order"][part].reshape(-1)].view(torch.float8_e4m3fn).float()
    c = c * state["scales"][table, :, part].float()[..., None]
    kvh = c.shape[1]
    return c.view(-1, kvh, 16, width)[..., :hd].transpose(0, 1).reshape(kvh, -1, hd)


def _attend(state):
    case = state["case"]
    qh, kvh, hd = SHAPES[case["shape"]]
    group = qh // kvh
    for (ctx, n, row), table in zip(_sessions(case), state["tables"]):
        k, v = (_values(state, table, part, hd)[:, : ctx + n] for part in range(2))
        q = state["q"][row: row + n].float().view(n, kvh, group, hd).permute(1, 2, 0, 3).reshape(kvh, group * n, hd)
        s = torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(hd)
        seen = torch.arange(ctx + n, device="cuda") <= ctx + torch.arange(n, device="cuda")[:, None]
        s = s.view(kvh, group, n, -1).masked_fill_(~seen, -math.inf)
        s = torch.exp(s - s.amax(-1, keepdim=True))
        s /= s.sum(-1, keepdim=True)
        o = torch.bmm(s.view(kvh, group * n, -1), v.contiguous())
        state["out"][row: row + n] = o.view(kvh, group, n, hd).permute(2, 0, 1, 3).reshape(n, -1)
    return {"out": state["out"]}


def run(state):
    case = state["case"]
    if own:
        if case["op"] == "append":
            state["batch"].append_rows(state["pool"], 0, state["args"])
            got = {"q": state["out"]} if case["rope"] else {}
        else:
            state["batch"].attention_rows(state["pool"], 0, state["args"])
            return {"out": state["out"]}
    elif case["op"] == "append":
        got = _append(state)
    else:
        return _attend(state)
    # the cache after the step: the codes as the numbers they are, and the blocks' powers of two
    return dict(got, codes=state["blocks"].view(torch.float8_e4m3fn), scales=state["scales"])


# ---------------------------------------------------------------------------
# The same in 64 bits
# ---------------------------------------------------------------------------
def _number(codes):
    """The value of e4m3 bits: sign, four exponent bits (bias 7), three of the mantissa."""
    u = codes.to(torch.int64)
    exp, man = (u >> 3) & 15, (u & 7).double()
    mag = torch.where(exp > 0, (8.0 + man) * 2.0 ** (exp - 10).double(), man * 2.0 ** -9)
    return torch.where(u > 127, -mag, mag)


def _where(width):
    """[part][token][dim] -> place in the block, counted out."""
    at = torch.empty((2, 16, width), dtype=torch.int64)
    for t in range(16):
        for d in range(width):
            lane, j = d % 64 // 16 * 16 + t, d // 64 * 16 + d % 16
            at[0, t, d] = j // 16 * 1024 + lane * 16 + j % 16
            lane, j = t // 4 * 16 + d % 16, (d % 32 // 16) * (width // 32) * 4 + d // 32 * 4 + t % 4
            at[1, t, d] = 16 * width + j // 16 * 1024 + lane * 16 + j % 16
    return at.to("cuda")


def exact(case, seed):
    qh, kvh, hd = SHAPES[case["shape"]]
    width = _block_width(hd)
    x = _inputs(case, seed)
    at = _where(width)
    if case["op"] == "attend":
        out = torch.empty((x["q"].shape[0], qh * hd), dtype=torch.float64, device="cuda")
        for (ctx, n, row), table in zip(_sessions(case), x["tables"]):
            bits, power = x["blocks"][table], x["scales"][table].double()
            pos = ctx + torch.arange(n, device="cuda")
            for head in range(kvh):
                kv = []
                for part in range(2):
                    val = _number(bits[:, head][:, at[part, :, :hd].reshape(-1)]) * power[:, head, part, None]
                    kv.append(val.reshape(-1, hd)[: ctx + n].contiguous())
                hidden = torch.arange(ctx + n, device="cuda")[None] > pos[:, None]
                for one in range(head * (qh // kvh), (head + 1) * (qh // kvh)):
                    cols = slice(one * hd, (one + 1) * hd)
                    s = x["q"][row: row + n, cols].double() @ kv[0].T.contiguous() * hd ** -0.5
                    s[hidden] = -math.inf
                    out[row: row + n, cols] = torch.softmax(s, -1) @ kv[1]
        return {"out": out}
    k, v, q = (x[name].double() for name in ("k", "v", "q"))
    got = {}
    if case["rope"]:
        pos = torch.cat([torch.arange(ctx, ctx + n, device="cuda") for ctx, n, _ in _sessions(case)])
        turn = torch.complex(x["cos"][pos].double(), x["sin"][pos].double())[:, None]

        def rotate(y, bias):
            y = (y + bias.double()).view(y.shape[0], -1, 2, hd // 2)
            z = torch.complex(y[:, :, 0].contiguous(), y[:, :, 1].contiguous()) * turn
            return torch.stack([z.real, z.imag], 2).reshape(y.shape[0], -1)

        q, k, v = rotate(q, x["q_bias"]), rotate(k, x["k_bias"]), v + x["v_bias"].double()
        got["q"] = q
    codes, scales = _number(x["blocks"]), x["scales"].double()
    for (ctx, n, row), table in zip(_sessions(case), x["tables"]):
        for part, rows in ((0, k), (1, v)):
            first = ctx // 16
            new = torch.zeros((kvh, (len(table) - first) * 16, hd), dtype=torch.float64, device="cuda")
            new[:, ctx - first * 16: ctx - first * 16 + n] = rows[row: row + n].view(n, kvh, hd).transpose(0, 1)
            new = new.view(kvh, -1, 16, hd).transpose(0, 1)  # [page][head][slot][dim]
            e = torch.ceil(torch.log2(new.abs().amax((-1, -2)) / 448.0)).clamp(-15, 7)
            if ctx % 16:
                e[0] = torch.maximum(e[0], torch.log2(scales[table[first], :, part]))
            place = at[part, :, :hd].reshape(-1)
            new = new * 2.0 ** -e[..., None, None]
            if ctx % 16:
                was = codes[table[first]][:, place].view(kvh, 16, hd)
                was = was * (scales[table[first], :, part] / 2.0 ** e[0])[:, None, None]
                new[0, :, : ctx % 16] = was[:, : ctx % 16]
            page = codes[table[first:]]
            page[:, :, place] = new.reshape(len(table) - first, kvh, 16 * hd)
            codes[table[first:]] = page
            scales[table[first:], :, part] = 2.0 ** e
    return dict(got, codes=codes, scales=scales)
