"""The e4m3 cache on the GPU against its 64-bit model: appends bit for bit,
attention within a bound derived from the kernel's roundings (_e4m3.attend)."""
import ctypes as C

import numpy as np
import pytest

import _e4m3 as M
import tge_kv as tk

pytestmark = pytest.mark.gpu

TYPES = [tk.ROWS_F32, tk.ROWS_F16, tk.ROWS_BF16]
SHAPES = [(14, 2, 64), (12, 2, 128), (28, 4, 128), (16, 8, 256), (16, 4, 96), (5, 5, 8), (9, 3, 72), (6, 2, 200),
          (7, 1, 248)]


def one_session(qh, kvh, hd, ctx, n, **more):
    return M.Case(qh, kvh, hd, [(ctx, n)], **more)


def append(case, rows, row_type, gap=0, layer=0):
    k = M.Rows(np.concatenate([r[0] for r in rows]), row_type, gap)
    v = M.Rows(np.concatenate([r[1] for r in rows]), row_type, gap)
    b = case.plan()
    b.append_rows(case.pool, layer, tk.append_rows_args(row_type, k, v, k_stride=k.stride, v_stride=v.stride))
    tk.hip().sync()
    for (c, _), cache, r in zip(case.sessions, case.cache, rows):
        cache.append(c, *r)
    return b


def attend(case, row_type, gap=0, scale=0.0, q_gain=1.0, batch=None, layer=0):
    """Runs the step's attention; returns (out, want, bound) rows of all sessions."""
    n = sum(n for _, n in case.sessions)
    q = M.as_type(case.rng.standard_normal((n, case.qh * case.hd)) * q_gain, row_type)
    dq = M.Rows(q, row_type, gap)
    out = M.Rows(np.zeros_like(q), row_type, gap, spare=3)
    b = batch or case.plan()
    b.attention_rows(case.pool, layer, tk.attention_rows_args(row_type, dq, out, q_stride=dq.stride,
                                                              out_stride=out.stride, scale=scale))
    tk.hip().sync()
    got = out.read()
    want, bound, row = [], [], 0
    for (c, m), cache in zip(case.sessions, case.cache):
        w, e = M.attend(cache, c, q[row: row + m], case.qh, scale or None)
        want.append(w)
        bound.append(e)
        row += m
    return got, np.concatenate(want), np.concatenate(bound)


def check(got, want, bound, row_type):
    # the output's own rounding: half a step of its value (subnormal f16: 2^-25)
    limit = bound + M.HALF_STEP[row_type] * (np.abs(want) + bound) + 2.0 ** -25
    worst = np.max(np.abs(got - want) / limit)
    assert np.isfinite(got).all() and worst <= 1.0, worst


# ---- append ------------------------------------------------------------------
def test_every_code_and_tie(gpu):
    """Values on codes, on ties and beside them over the whole range, with a
    448 in each block so that the scale is 1."""
    p = M.POSITIVE
    mid = (p[:-1] + p[1:]) / 2
    x = np.concatenate([p, mid, np.nextafter(np.float32(mid), np.float32(0)), np.nextafter(np.float32(mid), np.float32(1e9)),
                        [2.0 ** -11, 2.0 ** -10, 0.0, -0.0]]).astype(np.float32)
    x = np.concatenate([x, -x])
    x = np.concatenate([x, np.zeros(-len(x) % 127, np.float32)]).reshape(-1, 127)
    x = np.concatenate([x, np.full((len(x), 1), 448.0, np.float32)], 1)
    case = one_session(1, 1, 128, 0, len(x))
    b = append(case, [(x, -x)], tk.ROWS_F32)
    case.check_pool(b)
    assert (case.cache[0].exps[0] == 0).all()


@pytest.mark.parametrize("row_type", TYPES)
@pytest.mark.parametrize("qh,kvh,hd", SHAPES)
def test_append_bits(gpu, qh, kvh, hd, row_type):
    """Ragged sessions: pages begun before, written whole, ended in part; then
    further single tokens whose scales may grow."""
    case = M.Case(qh, kvh, hd, [(0, 1), (5, 3), (15, 2), (16, 16), (31, 50), (0, 33), (40, 1)], seed=hd + row_type)
    case.fill(row_type)
    b = append(case, case.step_rows(row_type), row_type, gap=8)
    case.check_pool(b)
    for step in range(3):
        case.sessions = [(len(c.codes[0]), 1) for c in case.cache]
        case.pages = [p + [case.table.allocate()] if len(p) * 16 <= c else p
                      for p, (c, _) in zip(case.pages, case.sessions)] if step == 0 else case.pages
        if any(len(p) * 16 <= c for p, (c, _) in zip(case.pages, case.sessions)):
            break
        rows = [(k * np.float32(3.0 ** step), v * np.float32(5.0 ** step)) for k, v in case.step_rows(tk.ROWS_F32)]
        b = append(case, rows, tk.ROWS_F32)
        case.check_pool(b)


def test_scale_grows_and_old_codes_follow(gpu):
    """A loud token moves the scale by up to 22 steps: the older codes are
    re-encoded, the smallest through subnormals to zero."""
    for gain in (1.9, 2.1, 40.0, 1e3, 1e5, 3e6):
        case = one_session(4, 2, 128, 11, 2, seed=int(gain), loud=False)
        case.fill()
        k, v = case.rows(2, tk.ROWS_F32)
        k[1, 3] = np.float32(448.0 * gain / 100)
        v[0, 200] = np.float32(-gain)
        b = append(case, [(k, v)], tk.ROWS_F32)
        case.check_pool(b)


def test_slots_behind_the_last_row_are_cleared(gpu):
    """A page that held other rows is taken anew, and rejected drafts go when
    the step after them is stored."""
    case = one_session(4, 2, 72, 0, 48)
    append(case, case.step_rows(tk.ROWS_F32), tk.ROWS_F32)
    case.sessions = [(3, 2)]
    cache = case.cache[0]
    cache.codes = [c[:3] for c in cache.codes]
    cache.exps = [e[:1] for e in cache.exps]
    b = append(case, case.step_rows(tk.ROWS_F32), tk.ROWS_F32)
    case.check_pool(b)
    codes, _ = M.raw_layer(case.pool)
    page = codes[case.pages[0][0]]
    live = np.zeros(page.shape[-1], bool)
    for part in range(2):
        live[:] = False
        for t in range(5):
            for d in range(72):
                live[tk.lib().tge_kv_e4m3_index(part, t, d, 128)] = True
        assert (page[:, part][:, ~live] == 0).all()


def test_extremes(gpu):
    """Infinities, NaN, the type's largest and smallest values, all zeros."""
    x = np.zeros((20, 64), np.float32)
    x[0, :8] = [np.inf, -np.inf, np.nan, 3.4e38, -3.4e38, 1e-45, -1e-38, 60000.0]
    x[16, :4] = [1e-45, np.nan, -0.0, 1e-30]
    case = one_session(1, 1, 64, 0, 20)
    b = append(case, [(x, -x)], tk.ROWS_F32)
    case.check_pool(b)
    assert case.cache[0].exps[0][0, 0] == 7 and case.cache[0].exps[0][1, 0] == -15


@pytest.mark.parametrize("fma", [True, False])
@pytest.mark.parametrize("row_type", TYPES)
@pytest.mark.parametrize("qh,kvh,hd", [(14, 2, 64), (28, 4, 128), (16, 8, 256), (6, 2, 48), (16, 4, 96), (4, 4, 80),
                                       (3, 3, 16), (2, 1, 208)])
def test_append_rotates(gpu, qh, kvh, hd, row_type, fma):
    case = M.Case(qh, kvh, hd, [(0, 5), (13, 4), (200, 40), (31, 1)], seed=hd + 7 * row_type)
    case.fill(row_type)
    rng = case.rng
    cos, sin = tk.rope_tables(hd, 241)
    n = sum(m for _, m in case.sessions)
    q = M.as_type(rng.standard_normal((n, qh * hd)), row_type)
    kv = case.step_rows(row_type)
    bias = [M.f32(rng.standard_normal(w)) for w in (qh * hd, kvh * hd, kvh * hd)]
    dk, dv = (M.Rows(np.concatenate([r[i] for r in kv]), row_type, 16) for i in (0, 1))
    dq, dqo = M.Rows(q, row_type, 8), M.Rows(np.zeros_like(q), row_type, 24, spare=2)
    db = [tk.DeviceArray.from_numpy(x) for x in bias]
    tabs = [tk.DeviceArray.from_numpy(x) for x in (cos, sin)]
    pos = np.concatenate([np.arange(c, c + m) for c, m in case.sessions])
    for in_place in (False, True):
        to = dq if in_place else dqo
        args = tk.append_rows_args(row_type, dk, dv, dk.stride, dv.stride, dq, to, dq.stride, to.stride, *db, *tabs,
                                   cos.shape[0], fma=fma)
        b = case.plan()
        b.append_rows(case.pool, 0, args)
        tk.hip().sync()
        want_q = M.as_type(M.rotate(q, bias[0], cos[pos], sin[pos], hd, fma), row_type)
        assert np.array_equal(to.read(), want_q)
    at = 0
    for (c, m), cache, (k, v) in zip(case.sessions, case.cache, kv):
        p = np.arange(c, c + m)
        cache.append(c, M.rotate(k, bias[1], cos[p], sin[p], hd, fma), M.f32(v + bias[2]))
        at += m
    case.check_pool(b)


# ---- attention -----------------------------------------------------------------
@pytest.mark.parametrize("row_type", TYPES)
@pytest.mark.parametrize("qh,kvh,hd", SHAPES)
def test_decode(gpu, qh, kvh, hd, row_type):
    """One new token, and drafted tokens, over ragged contexts."""
    for n in (1, 4):
        case = M.Case(qh, kvh, hd, [(0, n), (1, n), (14, n), (15, n), (16, n), (63, n), (400, n)], seed=hd + n)
        case.fill(row_type)
        append(case, case.step_rows(row_type), row_type)
        check(*attend(case, row_type, gap=8), row_type)


@pytest.mark.parametrize("qh,kvh,hd", [(28, 4, 128), (14, 2, 64), (16, 8, 256)])
def test_decode_long(gpu, qh, kvh, hd):
    """Contexts that are cut into several pieces and merged in the launch."""
    case = M.Case(qh, kvh, hd, [(9000, 2), (17, 1), (2500, 4)], seed=3)
    case.fill(tk.ROWS_BF16)
    b = append(case, case.step_rows(tk.ROWS_BF16), tk.ROWS_BF16)
    assert b.info()[2] > 1
    check(*attend(case, tk.ROWS_BF16, batch=b), tk.ROWS_BF16)
    # again on the same plan: the arrival counters are re-armed
    check(*attend(case, tk.ROWS_BF16, batch=b), tk.ROWS_BF16)


@pytest.mark.parametrize("row_type", TYPES)
@pytest.mark.parametrize("qh,kvh,hd,ctx,n", [
    (14, 2, 64, 0, 100), (12, 2, 128, 37, 65), (28, 4, 128, 100, 90), (16, 8, 256, 20, 70), (16, 4, 96, 0, 131),
    (64, 1, 128, 5, 9), (128, 1, 64, 3, 3), (64, 1, 256, 0, 5), (5, 5, 8, 0, 200), (6, 2, 200, 33, 50)])
def test_prompt(gpu, qh, kvh, hd, ctx, n, row_type):
    case = one_session(qh, kvh, hd, ctx, n, seed=hd + n)
    case.fill(row_type)
    append(case, case.step_rows(row_type), row_type)
    check(*attend(case, row_type, gap=16), row_type)


def test_prompt_split_and_wide_tiles(gpu):
    """A chunk late in a long context (pieces merged in the launch), and one
    with tiles of 128 rows (checked at every 37th row)."""
    case = one_session(8, 2, 128, 6000, 40, seed=5)
    case.fill(tk.ROWS_BF16)
    b = append(case, case.step_rows(tk.ROWS_BF16), tk.ROWS_BF16)
    assert b.info()[2] > 1
    check(*attend(case, tk.ROWS_BF16, batch=b), tk.ROWS_BF16)


def sampled(case, row_type, every):
    n = sum(m for _, m in case.sessions)
    q = M.as_type(case.rng.standard_normal((n, case.qh * case.hd)), row_type)
    dq, out = M.Rows(q, row_type), M.Rows(np.zeros_like(q), row_type)
    b = case.plan()
    b.attention_rows(case.pool, 0, tk.attention_rows_args(row_type, dq, out))
    tk.hip().sync()
    got, row = out.read(), 0
    for (c, m), cache in zip(case.sessions, case.cache):
        for i in range(0, m, every):
            want, bound = M.attend(cache, c + i, q[row + i: row + i + 1], case.qh)
            check(got[row + i: row + i + 1], want, bound, row_type)
        row += m


@pytest.mark.parametrize("qh,kvh,hd,ctx,n", [(28, 4, 128, 0, 1333), (32, 8, 64, 50, 1500), (16, 8, 256, 0, 2100)])
def test_prompt_large(gpu, qh, kvh, hd, ctx, n):
    case = one_session(qh, kvh, hd, ctx, n, seed=9)
    case.fill(tk.ROWS_BF16)
    append(case, case.step_rows(tk.ROWS_BF16), tk.ROWS_BF16)
    sampled(case, tk.ROWS_BF16, 37)


@pytest.mark.parametrize("qh,kvh,hd,ctx,n,sessions", M.LONG_ITEMS)
def test_long_items(gpu, qh, kvh, hd, ctx, n, sessions):
    """Items of more pages than the block numbers held at a time, many
    sessions over one session's pages (some rows checked)."""
    case = one_session(qh, kvh, hd, ctx, n, seed=35)
    case.fill(tk.ROWS_BF16)
    append(case, case.step_rows(tk.ROWS_BF16), tk.ROWS_BF16)
    rows = n * sessions
    q = M.as_type(case.rng.standard_normal((rows, qh * hd)), tk.ROWS_BF16)
    dq, out = M.Rows(q, tk.ROWS_BF16), M.Rows(np.zeros_like(q), tk.ROWS_BF16)
    b = case.plan([tk.Session(ctx, n, case.pages[0])] * sessions)
    b.attention_rows(case.pool, 0, tk.attention_rows_args(tk.ROWS_BF16, dq, out))
    tk.hip().sync()
    got = out.read()
    for i in (0, rows // 2, rows - 1):
        want, bound = M.attend(case.cache[0], ctx + i % n, q[i: i + 1], qh)
        check(got[i: i + 1], want, bound, tk.ROWS_BF16)


@pytest.mark.parametrize("qh,kvh,hd", [(28, 4, 128), (16, 8, 256), (14, 2, 64)])
def test_mixed(gpu, qh, kvh, hd):
    case = M.Case(qh, kvh, hd, [(300, 1), (40, 70), (0, 3), (513, 4), (7, 100)], seed=11)
    case.fill(tk.ROWS_F16)
    append(case, case.step_rows(tk.ROWS_F16), tk.ROWS_F16)
    check(*attend(case, tk.ROWS_F16, gap=8), tk.ROWS_F16)


def test_scale_and_peaked_rows(gpu):
    """A given softmax scale, and scores whose spread passes the lazy base."""
    case = M.Case(8, 2, 128, [(700, 3), (33, 70)], seed=13)
    case.fill(tk.ROWS_F32)
    append(case, case.step_rows(tk.ROWS_F32), tk.ROWS_F32)
    check(*attend(case, tk.ROWS_BF16, scale=0.031), tk.ROWS_BF16)
    check(*attend(case, tk.ROWS_F32, q_gain=12.0), tk.ROWS_F32)


def test_small_values_reach_the_matrix_cores(gpu):
    """K and V whose stored values are subnormal in f16."""
    case = one_session(4, 2, 128, 0, 40, seed=15, loud=False)
    rows = [(k * np.float32(2.0 ** -18), v * np.float32(2.0 ** -18)) for k, v in case.step_rows(tk.ROWS_F32)]
    append(case, rows, tk.ROWS_F32)
    got, want, bound = attend(case, tk.ROWS_F32, q_gain=1000.0)
    limit = bound + 2.0 ** -24 * np.abs(want)
    assert np.max(np.abs(want)) > 2.0 ** -19 and (np.abs(got - want) <= limit).all()


def test_nan_rows_stay_alone(gpu):
    """A NaN in one q row reaches that row and head only; NaN and infinite K
    and V rows are stored finite, so rows before them stay clean."""
    case = one_session(4, 2, 64, 20, 30, seed=17)
    case.fill()
    rows = case.step_rows(tk.ROWS_F32)
    rows[0][0][20, 5] = np.nan
    rows[0][1][21, :] = np.nan
    append(case, rows, tk.ROWS_F32)
    q = M.f32(case.rng.standard_normal((30, 4 * 64)))
    q[7, 64 + 3] = np.nan
    dq, out = M.Rows(q, tk.ROWS_F32), M.Rows(np.zeros_like(q), tk.ROWS_F32)
    case.plan().attention_rows(case.pool, 0, tk.attention_rows_args(tk.ROWS_F32, dq, out))
    tk.hip().sync()
    got = out.read()
    bad = np.isnan(got)
    assert bad[7, 64:128].all()
    bad[7, 64:128] = False
    assert not bad.any()


@pytest.mark.parametrize("row_type", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_infinite_queries_give_nan(gpu, hd, row_type):
    """A row whose q holds an infinity (or, scaled, a value past f16's largest)
    is NaN whether its scores are all +inf or all -inf; the rows around it are
    what they are without it. One visible position, a part of a page, a context
    in pieces, a prompt."""
    qh, kvh, bad = 4, 2, 3
    case = M.Case(qh, kvh, hd, [(0, 1), (40, 2), (9000, 2), (5, 70)], seed=hd)
    plain = case.rows

    def rows(n, t):  # (dim `bad` of every K row is positive)
        k, v = plain(n, t)
        k[:, bad::hd] = M.as_type(np.abs(k[:, bad::hd]) + 1.0, t)
        return k, v

    case.rows = rows
    case.fill(row_type)
    b = append(case, case.step_rows(row_type), row_type)
    assert b.info()[2] > 1
    n = sum(m for _, m in case.sessions)
    q = M.as_type(case.rng.standard_normal((n, qh * hd)), row_type)
    past = np.inf if row_type == tk.ROWS_F16 else 1e7
    want_nan = np.zeros((n, qh), bool)
    sent = q.copy()
    for i in range(n):
        for h in range(qh):
            if (i + h) % 3 == 0:
                want_nan[i, h] = True
                sent[i, h * hd + bad] = [np.inf, -np.inf, past, -past][(i // 3 + h) % 4]
    dq, out = M.Rows(sent, row_type), M.Rows(np.zeros_like(q), row_type)
    b.attention_rows(case.pool, 0, tk.attention_rows_args(row_type, dq, out))
    tk.hip().sync()
    got, row = out.read().reshape(n, qh, hd), 0
    assert np.isnan(got[want_nan]).all(), np.argwhere(want_nan & ~np.isnan(got).all(-1))
    for (c, m), cache in zip(case.sessions, case.cache):
        want, bound = (x.reshape(m, qh, hd) for x in M.attend(cache, c, q[row: row + m], qh))
        live = ~want_nan[row: row + m]
        check(got[row: row + m][live], want[live], bound[live], row_type)
        row += m


def test_stale_pages_do_not_reach_a_row(gpu):
    """Every byte of the pool is a NaN code before the step is stored."""
    case = M.Case(8, 2, 128, [(0, 5), (0, 33)], seed=19)
    view = case.pool.layer(0)
    tk.hip().memset(view.k, 0x7F, case.pool.bytes())
    append(case, case.step_rows(tk.ROWS_F32), tk.ROWS_F32)
    check(*attend(case, tk.ROWS_F32), tk.ROWS_F32)


# ---- the calls together ------------------------------------------------------------
def test_fp32_calls_and_layers(gpu):
    """The fp32 entry points on an e4m3 pool run the same kernels; layers are apart."""
    case = M.Case(12, 2, 128, [(50, 2), (9, 3)], seed=21, layers=3)
    case.fill(layer=1)
    k, v = (np.concatenate(x) for x in zip(*case.step_rows(tk.ROWS_F32)))
    q = M.f32(case.rng.standard_normal((5, 12 * 128)))
    dk, dv, dq = (tk.DeviceArray.from_numpy(x) for x in (k, v, q))
    outs = [tk.DeviceArray(q.shape, np.float32).zero() for _ in range(5)]
    b = case.plan()
    b.append(case.pool, 1, dk, dv)
    b.decode(case.pool, 1, dq, outs[0])
    b.decode_step(case.pool, 1, dq, dk, dv, outs[1])
    b.attention(case.pool, 1, dq, outs[2])
    b.prefill(case.pool, 1, dq, outs[3])
    b.attention_rows(case.pool, 1, tk.attention_rows_args(tk.ROWS_F32, dq, outs[4]))
    tk.hip().sync()
    got = [o.numpy() for o in outs]
    assert all(np.array_equal(got[0], g) for g in got[1:])
    row = 0
    for (c, n), cache in zip(case.sessions, case.cache):
        cache.append(c, k[row: row + n], v[row: row + n])
        want, bound = M.attend(cache, c, q[row: row + n], 12)
        check(got[0][row: row + n], want, bound, tk.ROWS_F32)
        row += n
    case.check_pool(b, 1)
    codes, scales = M.raw_layer(case.pool, 0)
    assert not codes.any() and not scales.any()
    codes, scales = M.raw_layer(case.pool, 2)
    assert not codes.any() and not scales.any()


def test_copy_page(gpu):
    case = M.Case(4, 2, 64, [(20, 4)], seed=23, layers=2)
    case.fill(layer=0)
    append(case, case.step_rows(tk.ROWS_F32), tk.ROWS_F32)
    free = case.table.allocate()
    case.pool.copy_page(case.pages[0][1], free)
    codes, scales = M.raw_layer(case.pool, 0)
    assert np.array_equal(codes[free], codes[case.pages[0][1]]) and codes[free].any()
    assert np.array_equal(scales[free], scales[case.pages[0][1]])


def test_copy_page_in_every_layer(gpu):
    """Codes and scales of the page in each layer, and nothing else."""
    case = M.Case(6, 3, 64, [(20, 4)], seed=45, layers=3)
    for layer in range(3):
        case.cache = [M.Cache(3, 64)]
        case.fill(layer=layer)
        rows = [(k * np.float32(4.0 ** layer), v) for k, v in case.step_rows(tk.ROWS_F32)]
        append(case, rows, tk.ROWS_F32, layer=layer)
    free = case.table.allocate()
    before = [M.raw_layer(case.pool, layer) for layer in range(3)]
    source = case.pages[0][1]
    case.pool.copy_page(source, free)
    for layer, (codes, scales) in enumerate(before):
        codes[free], scales[free] = codes[source], scales[source]
        got = M.raw_layer(case.pool, layer)
        assert np.array_equal(got[0], codes) and np.array_equal(got[1], scales), layer
        assert codes[free].any() and scales[free].any()
    # (the layers' pages differ, so that one layer's copy cannot pass for another's)
    assert not np.array_equal(before[0][1][source], before[1][1][source])
    assert not np.array_equal(before[1][1][source], before[2][1][source])


def test_driver_serves_16_bit_rows(gpu):
    """The Qwen2-shaped driver over steps of a session: prompt, decode, drafts
    that are rejected, decode again, every step against the model."""
    qh, kvh, hd, layers = 12, 2, 128, 2
    m = tk.Qwen2KvPath(layers, qh, kvh, hd, context=512, sequences=2, pages=80, fmt=tk.KV_E4M3)
    m.table().fragment(5)
    rng = np.random.default_rng(25)
    cos, sin = tk.rope_tables(hd, 512)
    tabs = [tk.DeviceArray.from_numpy(x) for x in (cos, sin)]
    caches = [[M.Cache(kvh, hd) for _ in range(layers)] for _ in range(2)]
    t = tk.ROWS_BF16
    for seq, start, n in [(0, 0, 90), (1, 0, 20), (0, 90, 1), (0, 91, 5), (0, 93, 1), (1, 20, 3), (0, 94, 70)]:
        if n == 1:
            m.begin_forward(seq, start)
        else:
            m.begin_prefill(seq, start, n)
        pos = np.arange(start, start + n)
        for layer in range(layers):
            fused = M.as_type(rng.standard_normal((n, (qh + 2 * kvh) * hd)), t)
            buf = M.Rows(fused, t)
            rot, out = M.Rows(np.zeros((n, qh * hd)), t), M.Rows(np.zeros((n, qh * hd)), t, spare=1)
            store = tk.append_rows_args(t, buf.ptr + 2 * qh * hd, buf.ptr + 2 * (qh + kvh) * hd, buf.stride, buf.stride,
                                        buf.ptr, rot, buf.stride, rot.stride, rope_cos=tabs[0], rope_sin=tabs[1],
                                        rope_positions=512)
            m.layer_rows(layer, store, tk.attention_rows_args(t, rot, out))
            tk.hip().sync()
            q, k, v = np.split(fused, [qh * hd, (qh + kvh) * hd], 1)
            cache = caches[seq][layer]
            cache.append(start, M.rotate(k, np.zeros(kvh * hd), cos[pos], sin[pos], hd), v)
            q = M.as_type(M.rotate(q, np.zeros(qh * hd), cos[pos], sin[pos], hd), t)
            assert np.array_equal(rot.read(), q)
            check(out.read(), *M.attend(cache, start, q, qh), t)
    m.close()


def test_driver_shares_and_copies_pages(gpu):
    """A sequence takes over 47 of another's 50 tokens and writes its own behind
    them: the page that both hold is copied, codes and scales, and neither sees
    the other's rows afterwards."""
    qh, kvh, hd, t = 8, 2, 128, tk.ROWS_BF16
    m = tk.Qwen2KvPath(1, qh, kvh, hd, context=256, sequences=2, pages=40, fmt=tk.KV_E4M3)
    rng = np.random.default_rng(37)
    caches = [M.Cache(kvh, hd), M.Cache(kvh, hd)]

    def step(seq, start, n):
        if n == 1:
            m.begin_forward(seq, start)
        else:
            m.begin_prefill(seq, start, n)
        q, k, v = (M.as_type(rng.standard_normal((n, h * hd)) * (1 + start), t) for h in (qh, kvh, kvh))
        rows = [M.Rows(x, t) for x in (q / np.float32(1 + start), k, v)]
        out = M.Rows(np.zeros((n, qh * hd)), t)
        m.layer_rows(0, tk.append_rows_args(t, *rows[1:]), tk.attention_rows_args(t, rows[0], out))
        tk.hip().sync()
        caches[seq].append(start, k, v)
        check(out.read(), *M.attend(caches[seq], start, rows[0].read(), qh), t)

    tokens = list(range(100, 150))
    step(0, 0, 50)
    assert m.remember_prefix(0, tokens) == 50
    assert m.attach_prefix(1, tokens[:47] + [5] * 20) == 47
    caches[1].codes = [c[:47].copy() for c in caches[0].codes]
    caches[1].exps = [e[:3].copy() for e in caches[0].exps]
    step(1, 47, 20)  # (louder rows: the copy's scales and older codes change)
    step(0, 50, 1)
    step(1, 67, 1)
    m.close()


def test_repeatable_and_independent_of_the_pages(gpu):
    """Bit-identical on every run, wherever the pages sit."""
    got = []
    for seed in (27, 27, 28):
        case = M.Case(28, 4, 128, [(3000, 4), (700, 1), (90, 80)], seed=27)
        case.table.close()
        if seed == 28:  # the same rows in other pages
            ids = [p for ps in case.pages for p in ps]
            other = iter(np.random.default_rng(1).permutation(ids).tolist())
            case.pages = [[next(other) for _ in ps] for ps in case.pages]
        case.fill(tk.ROWS_BF16)
        append(case, case.step_rows(tk.ROWS_BF16), tk.ROWS_BF16)
        q = M.Rows(M.as_type(np.random.default_rng(2).standard_normal((85, 28 * 128)), tk.ROWS_BF16), tk.ROWS_BF16)
        for _ in range(2):
            out = M.Rows(np.zeros((85, 28 * 128)), tk.ROWS_BF16)
            case.plan().attention_rows(case.pool, 0, tk.attention_rows_args(tk.ROWS_BF16, q, out))
            tk.hip().sync()
            got.append(out.read())
        case.close()
    assert all(np.array_equal(got[0], g) for g in got[1:])


def test_captured_calls_replay(gpu):
    """Append and attention of a step in a graph on a stream of its own:
    every replay takes the buffers' present contents."""
    h = tk.hip().h
    case = M.Case(12, 2, 128, [(2000, 2), (30, 1), (10, 40)], seed=29)
    case.fill(tk.ROWS_BF16)
    t, n = tk.ROWS_BF16, 43
    st = C.c_void_p()
    tk.hip().ok(h.hipStreamCreate(C.byref(st)), "stream")
    k, v, q, out = (M.Rows(np.zeros((n, w)), t) for w in (256, 256, 12 * 128, 12 * 128))
    b = tk.Batch().plan(case.pool, [tk.Session(c, m, p) for (c, m), p in zip(case.sessions, case.pages)], 12, st)
    tk.hip().sync()
    graph, run = C.c_void_p(), C.c_void_p()
    tk.hip().ok(h.hipStreamBeginCapture(st, 0), "begin")
    b.append_rows(case.pool, 0, tk.append_rows_args(t, k, v), st)
    b.attention_rows(case.pool, 0, tk.attention_rows_args(t, q, out), st)
    with pytest.raises(tk.TgeError) as e:
        tk.Batch().plan(case.pool, [tk.Session(0, 1, case.pages[0])], 12, st)
    assert e.value.status == tk.ERR_INVALID
    tk.hip().ok(h.hipStreamEndCapture(st, C.byref(graph)), "end")
    tk.hip().ok(h.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)), "instantiate")
    before = [(list(c.codes), list(c.exps)) for c in case.cache]
    grown = None
    for replay in range(4):
        rows = [(kk * np.float32(0.5 + replay), vv) for kk, vv in case.step_rows(tk.ROWS_F32)]
        rows = [(M.as_type(a, t), M.as_type(c, t)) for a, c in rows]
        qq = M.as_type(case.rng.standard_normal((n, 12 * 128)), t)
        for dst, src in ((k, np.concatenate([r[0] for r in rows])), (v, np.concatenate([r[1] for r in rows])), (q, qq)):
            tk.hip().upload(dst.ptr, M.to_bytes(src, t))
        tk.hip().sync()
        tk.hip().ok(h.hipGraphLaunch(run, st), "launch")
        tk.hip().sync()
        got, row = out.read(), 0
        for s, ((c, m), cache, r) in enumerate(zip(case.sessions, case.cache, rows)):
            # (the step is stored again over the same slots: the older rows keep
            # what the earlier replays made of them)
            cache.append(c, *r)
            want, bound = M.attend(cache, c, qq[row: row + m], 12)
            check(got[row: row + m], want, bound, t)
            row += m
        case.check_pool(b)
    tk.hip().ok(h.hipGraphExecDestroy(run), "destroy")
    tk.hip().ok(h.hipGraphDestroy(graph), "destroy")
    tk.hip().ok(h.hipStreamDestroy(st), "destroy")


def test_captured_wide_attention_replays(gpu):
    """256-dim blocks size their LDS at the launch: captured, too."""
    h = tk.hip().h
    case = M.Case(16, 8, 256, [(900, 1), (40, 3)], seed=39)
    case.fill(tk.ROWS_F16)
    append(case, case.step_rows(tk.ROWS_F16), tk.ROWS_F16)
    q, out = (M.Rows(np.zeros((4, 16 * 256)), tk.ROWS_F16) for _ in range(2))
    b, st, graph, run = case.plan(), C.c_void_p(), C.c_void_p(), C.c_void_p()
    tk.hip().ok(h.hipStreamCreate(C.byref(st)), "stream")
    tk.hip().sync()
    tk.hip().ok(h.hipStreamBeginCapture(st, 0), "begin")
    b.attention_rows(case.pool, 0, tk.attention_rows_args(tk.ROWS_F16, q, out), st)
    tk.hip().ok(h.hipStreamEndCapture(st, C.byref(graph)), "end")
    tk.hip().ok(h.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)), "instantiate")
    for _ in range(3):
        x = M.as_type(case.rng.standard_normal((4, 16 * 256)), tk.ROWS_F16)
        tk.hip().upload(q.ptr, M.to_bytes(x, tk.ROWS_F16))
        tk.hip().sync()
        tk.hip().ok(h.hipGraphLaunch(run, st), "launch")
        tk.hip().sync()
        got = out.read()
        for rows, cache, ctx in ((slice(0, 1), case.cache[0], 900), (slice(1, 4), case.cache[1], 40)):
            check(got[rows], *M.attend(cache, ctx, x[rows], 16), tk.ROWS_F16)
    tk.hip().ok(h.hipGraphExecDestroy(run), "destroy")
    tk.hip().ok(h.hipGraphDestroy(graph), "destroy")
    tk.hip().ok(h.hipStreamDestroy(st), "destroy")


@pytest.mark.parametrize("qh,kvh,hd", [(28, 4, 128), (16, 8, 256), (14, 2, 64)])
def test_two_batches_on_two_streams(gpu, qh, kvh, hd):
    """Steps of two batches overlap: each has its own workspace."""
    h, t = tk.hip().h, tk.ROWS_BF16
    sides = []
    for seed, sessions in ((41, [(5000, 2), (100, 1)]), (43, [(3000, 1), (10, 70)])):
        case = M.Case(qh, kvh, hd, sessions, seed=seed)
        case.fill(t)
        append(case, case.step_rows(t), t)
        n = sum(m for _, m in sessions)
        q = M.as_type(case.rng.standard_normal((n, qh * hd)), t)
        st = C.c_void_p()
        tk.hip().ok(h.hipStreamCreate(C.byref(st)), "stream")
        b = tk.Batch().plan(case.pool, [tk.Session(c, m, p) for (c, m), p in zip(case.sessions, case.pages)], qh, st)
        sides.append((case, q, M.Rows(q, t), [M.Rows(np.zeros_like(q), t) for _ in range(4)], b, st))
    tk.hip().sync()
    for i in range(4):
        for case, _, q, outs, b, st in sides:
            b.attention_rows(case.pool, 0, tk.attention_rows_args(t, q, outs[i]), st)
    tk.hip().sync()
    for case, q, _, outs, _, st in sides:
        row = 0
        got = [o.read() for o in outs]
        assert all(np.array_equal(got[0], g) for g in got[1:])
        for (c, m), cache in zip(case.sessions, case.cache):
            check(got[0][row: row + m], *M.attend(cache, c, q[row: row + m], qh), t)
            row += m
        tk.hip().ok(h.hipStreamDestroy(st), "destroy")


def test_layer_past_4_gib(gpu):
    """A session whose pages sit past the 4 GiB mark of a layer's blocks."""
    pages = 530000  # x 2 heads x 4096 B
    pool = tk.KvPool(1, pages, 2, 128, tk.KV_E4M3)
    case = M.Case(4, 2, 128, [(300, 3)], seed=31)
    case.pool.close()
    case.pool = pool
    case.pages = [[pages - 1 - 3 * i for i in range(19)]]
    case.fill(tk.ROWS_BF16)
    b = append(case, case.step_rows(tk.ROWS_BF16), tk.ROWS_BF16)
    case.check_pool(b)
    check(*attend(case, tk.ROWS_BF16, batch=b), tk.ROWS_BF16)
    pool.close()


# ---- refusals ------------------------------------------------------------------------
def test_refusals(gpu):
    case = M.Case(4, 2, 64, [(20, 2), (3, 1)], seed=33)
    case.fill()
    before = M.raw_layer(case.pool)
    x = M.Rows(np.ones((3, 4 * 64 + 64)), tk.ROWS_F32)
    out = M.Rows(np.ones((3, 4 * 64)), tk.ROWS_F32)
    tab = tk.DeviceArray.from_numpy(np.zeros((22, 32), np.float32))
    b = case.plan()
    f16 = tk.KvPool(1, 8, 2, 64, tk.KV_F16)
    bf = tk.Batch().plan(f16, [tk.Session(0, 1, [0])], 4)
    t = tk.ROWS_F32

    def refused(call, *args):
        with pytest.raises(tk.TgeError) as e:
            call(*args)
        assert e.value.status == tk.ERR_INVALID, e.value

    def app(**more):
        a = dict(row_type=t, k=x.ptr, v=x.ptr)
        a.update(more)
        return tk.append_rows_args(**a)

    rope = dict(rope_cos=tab, rope_sin=tab, rope_positions=22)
    bad_append = [
        app(row_type=3), app(row_type=-1), app(k=None), app(v=None), app(k=x.ptr + 4), app(v=x.ptr + 8),
        app(k_stride=64), app(k_stride=-128), app(v_stride=130), app(row_type=tk.ROWS_BF16, k_stride=132),
        app(q=x.ptr, q_out=out.ptr), app(k_bias=x.ptr), app(rope_cos=tab), app(rope_sin=tab),
        app(**rope, q=x.ptr), app(**rope, q_out=out.ptr), app(**dict(rope, rope_positions=21)),
        app(**dict(rope, rope_cos=tab.ptr + 4)), app(**rope, v_bias=x.ptr + 8),
        app(**rope, q=x.ptr, q_out=x.ptr, q_stride=320), app(**rope, q=x.ptr + 4, q_out=out.ptr)]
    for a in bad_append:
        refused(b.append_rows, case.pool, 0, a)
    refused(b.append_rows, case.pool, 1, app())
    refused(b.append_rows, case.pool, -1, app())
    refused(bf.append_rows, f16, 0, app())
    refused(bf.attention_rows, f16, 0, tk.attention_rows_args(t, x, out))
    refused(b.append_rows, f16, 0, app())
    for a in [dict(row_type=9), dict(q=None), dict(out=None), dict(q=x.ptr + 4), dict(out=out.ptr + 8),
              dict(q_stride=64), dict(out_stride=258), dict(scale=-1.0), dict(scale=float("nan")),
              dict(scale=float("inf"))]:
        args = dict(row_type=t, q=x.ptr, out=out.ptr)
        args.update(a)
        refused(b.attention_rows, case.pool, 0, tk.attention_rows_args(**args))
    sparse = case.plan().set_sparse(4, 32, 2)
    refused(sparse.attention_rows, case.pool, 0, tk.attention_rows_args(t, x, out))
    refused(tk.decode_attention_static, case.pool, [tk.Session(20, 2, case.pages[0])], 4, 0, x, out)
    refused(lambda: tk.attention_group(case.pool, 0, 0, case.pages[0], 0, 4, np.zeros((2, 64), np.float32)))
    twice = tk.Batch().plan(case.pool, [tk.Session(0, 1, [0]), tk.Session(3, 1, [0])], 4)
    refused(twice.append_rows, case.pool, 0, app())
    refused(case.plan([tk.Session(0, 40, case.pages[0] + [case.table.allocate()])]).decode, case.pool, 0, x, out)
    codes, scales = M.raw_layer(case.pool)
    assert np.array_equal(codes, before[0]) and np.array_equal(scales, before[1])
    assert np.array_equal(out.read(), np.ones((3, 256), np.float32))
