"""Attention steps on an e4m3 pool by the kernel path that their plans take.

A session's pages are drawn, with repeats, from one stored sequence of
BASE_PAGES pages, so that long contexts and many tables cost one append."""
import math

import numpy as np

import _e4m3 as M
import tge_kv as tk

BASE_PAGES = 256


def ragged(count, longest, n_new, seed=5):
    """`count` sessions of contexts between 500 and `longest`, even in their logarithm."""
    rng = np.random.default_rng(seed)
    return [(int(math.exp(rng.uniform(math.log(500), math.log(longest)))), n_new) for _ in range(count)]


# name: (query heads, KV heads, head_dim, row type, sessions (ctx, new tokens), what the plan holds: keys of
# plan_e4m3_shape that are not 0, all others among rw1, rw2, rw4, chained, cut and outgrown being 0)
STEPS = {
    "serving": (28, 4, 128, tk.ROWS_BF16, ragged(64, 30000, 4), {"rw1", "chained", "unlike", "cut"}),
    "serving, 256 dims": (16, 8, 256, tk.ROWS_F16, ragged(32, 12000, 1), {"rw1", "chained", "unlike", "cut"}),
    "64 rows a head": (64, 8, 128, tk.ROWS_F16, ragged(40, 12000, 8), {"rw2", "chained", "unlike", "cut"}),
    "64 rows a head, 256 dims": (32, 4, 256, tk.ROWS_BF16, ragged(40, 12000, 8), {"rw2", "chained", "unlike", "cut"}),
    "mixed, 64 dims": (14, 2, 64, tk.ROWS_F32, ragged(64, 30000, 4, seed=6) + [(6000, 1000)],
                       {"rw1", "rw2", "chained", "unlike", "cut"}),
    "mixed": (28, 4, 128, tk.ROWS_F16, ragged(64, 12000, 4) + [(6000, 1000)], {"rw1", "rw4", "chained", "unlike", "cut"}),
    "mixed, 256 dims": (32, 4, 256, tk.ROWS_F32, ragged(40, 12000, 8) + [(12000, 900)],
                        {"rw2", "rw4", "chained", "unlike", "cut"}),
    "prompt in shares": (28, 4, 128, tk.ROWS_BF16, [(6000, 1000)], {"rw4", "chained", "cut"}),
    "prompt in shares, 64 dims": (128, 1, 64, tk.ROWS_BF16, [(8000, 700)], {"rw4", "chained", "cut"}),
    "prompt, 256 dims": (64, 1, 256, tk.ROWS_BF16, [(0, 1500)], {"rw4"}),
    "many pieces, 64 dims": (32, 1, 64, tk.ROWS_F32, [(90000, 1)], {"rw1", "cut", "outgrown"}),
    "many pieces of 64 rows": (64, 1, 64, tk.ROWS_BF16, [(90000, 1)], {"rw2", "cut", "outgrown"}),
    "many pieces": (64, 1, 128, tk.ROWS_F16, [(200000, 1)], {"rw2", "cut", "outgrown"}),
}
NOT_OTHERWISE = {"rw1", "rw2", "rw4", "chained", "cut", "outgrown"}


class Step:
    """The step's pool, tables and inputs. Scores spread widely, so that a row
    rests on few positions and a page that is missing, twice or another one
    shows in the rows that rest on it."""

    def __init__(self, name, gain=4.0):
        self.qh, self.kvh, self.hd, self.type, self.sessions, _ = STEPS[name]
        self.case = M.Case(self.qh, self.kvh, self.hd, [(BASE_PAGES * 16, 1)], seed=len(name), loud=False)
        self.case.fill(tk.ROWS_BF16)
        self.rng = np.random.default_rng(len(STEPS) + self.hd)
        self.tables = [self.rng.integers(0, BASE_PAGES, (c + n + 15) // 16) for c, n in self.sessions]
        ids = np.array(self.case.pages[0])
        self.batch = tk.Batch().plan(
            self.case.pool, [tk.Session(c, n, ids[t].tolist()) for (c, n), t in zip(self.sessions, self.tables)], self.qh)
        self.q = M.as_type(self.rng.standard_normal((sum(n for _, n in self.sessions), self.qh * self.hd)) * gain,
                           self.type)

    def run(self):
        q, out = M.Rows(self.q, self.type, gap=8), M.Rows(np.zeros_like(self.q), self.type, gap=16, spare=2)
        self.batch.attention_rows(self.case.pool, 0, tk.attention_rows_args(self.type, q, out, q.stride, out.stride))
        tk.hip().sync()
        return out.read()

    def checks(self, rows, heads=2):
        """(session, row of the step, columns, want, bound) of `rows` new tokens of
        each session, `heads` query heads of every KV head."""
        base, group, first = self.case.cache[0], self.qh // self.kvh, 0
        for s, ((ctx, n), table) in enumerate(zip(self.sessions, self.tables)):
            at = (table[:, None] * 16 + np.arange(16)).reshape(-1)
            # (the first token, the last, and others)
            take = sorted({0, n - 1, *self.rng.integers(0, n, max(rows - 2, 0)).tolist()} if rows > 1 else {n - 1})
            for h in range(self.kvh):
                one = M.Cache(1, self.hd)
                one.codes = [c[at, h: h + 1] for c in base.codes]
                one.exps = [e[table, h: h + 1] for e in base.exps]
                pick = h * group + self.rng.permutation(group)[:heads]
                cols = (pick[:, None] * self.hd + np.arange(self.hd)).reshape(-1)
                for i in take:
                    cut = M.Cache(1, self.hd)
                    need = (ctx + i) // 16 + 1
                    cut.codes, cut.exps = [c[: need * 16] for c in one.codes], [e[:need] for e in one.exps]
                    want, bound = M.attend(cut, ctx + i, self.q[first + i: first + i + 1, cols], len(pick))
                    yield s, first + i, cols, want[0], bound[0]
            first += n

    def close(self):
        self.case.close()
