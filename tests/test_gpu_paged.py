"""The paged K/V cache operators (include/itts_paged.h) on a B200 against plain
implementations: the bookkeeping against Python integers, the append against
torch's own rounding, the attention against its definition in 64 bits."""
import importlib
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def paged():
    return importlib.import_module("index-tts-25-metal_b200.paged")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---- tables -------------------------------------------------------------------


def plain_tables(cached, fresh, table, free, count, bs, blocks, rows):
    """The step's bookkeeping in Python integers; None where a status bit is due."""
    table, free = [list(r) for r in table], list(free)
    for b, f in enumerate(fresh):
        if f < 0:
            for j in range((cached[b] + bs - 1) // bs):
                free[count] = table[b][j]
                count += 1
    lens, q_start, positions, slots = [], [0], [], []
    for b, f in enumerate(fresh):
        n = max(f, 0)
        lens.append(0 if f < 0 else cached[b] + n)
        q_start.append(q_start[-1] + n)
        for p in range(cached[b], cached[b] + n):
            if p % bs == 0:
                count -= 1
                table[b][p // bs] = free[count]
            positions.append(p)
            slots.append(table[b][p // bs] * bs + p % bs)
    pad = rows - len(slots)
    return table, free, count, lens, q_start, positions + [0] * pad, slots + [-1] * pad


class TableState:
    def __init__(self, cached, fresh, bs, spare=0, rows=None, columns=None, seed=0):
        g = torch.Generator().manual_seed(seed)
        held = [(c + bs - 1) // bs for c in cached]
        need = [0 if f < 0 else (c + f + bs - 1) // bs - h for c, f, h in zip(cached, fresh, held)]
        given = sum(h for h, f in zip(held, fresh) if f < 0)
        self.columns = columns or max(1, max(h + n for h, n in zip(held, need)))
        self.blocks = max(1, sum(held) + max(0, sum(need) - given) + spare)
        ids = torch.randperm(self.blocks, generator=g).tolist()
        self.table = [[-7] * self.columns for _ in cached]
        for b, h in enumerate(held):
            self.table[b][:h] = [ids.pop() for _ in range(h)]
        self.count = len(ids)
        self.free = ids + [-9] * (self.blocks - len(ids))
        self.cached, self.fresh, self.bs = cached, fresh, bs
        self.rows = sum(max(f, 0) for f in fresh) if rows is None else rows

    def device(self):
        n = len(self.cached)
        return {"cached": ints(self.cached), "fresh": ints(self.fresh), "table": ints(self.table),
                "free_list": ints(self.free), "free_count": ints([self.count]), "lens": ints([99] * n),
                "q_start": ints([99] * (n + 1)), "positions": ints([99] * self.rows), "slots": ints([99] * self.rows),
                "status": ints([99]), "free_out": ints([99])}

    def check(self, d):
        want = plain_tables(self.cached, self.fresh, self.table, self.free, self.count, self.bs, self.blocks,
                            self.rows)
        assert d["status"].item() == 0
        got = [d[k].tolist() for k in ("table", "free_list", "free_out", "lens", "q_start", "positions", "slots")]
        assert got[0] == want[0] and got[1] == want[1] and got[2] == [want[2]] and got[3:] == list(want[3:])


def run_tables(paged, d, bs):
    kw = {k: d[k] for k in ("lens", "q_start", "positions", "slots", "status", "free_out")}
    paged.tables(d["cached"], d["fresh"], d["table"], d["free_list"], d["free_count"], bs, **kw)


TABLE_CASES = {
    "one": ([0], [1]),
    "one_none": ([5], [0]),
    "one_released": ([33], [-1]),
    "empty_released": ([0, 0, 3], [-1, 0, 1]),
    "edges": ([15, 16, 17, 0, 31, 32], [1, 1, 1, 16, 17, 0]),
    "all_released": ([7, 100, 16], [-1, -5, -2147483648]),
    "reuse": ([64, 0, 48, 0], [-1, 100, -1, 12]),
    "prompt": ([0], [5000]),
    "many": ([(37 * i) % 300 for i in range(700)], [(1 if i % 5 else (i * 13) % 90 if i % 2 else -1) for i in range(700)]),
    "wide": ([(11 * i) % 70 for i in range(8192)], [(i % 3) - 1 if i % 7 else i % 40 for i in range(8192)]),
}


@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("name", TABLE_CASES)
def test_tables(paged, name, bs):
    s = TableState(*TABLE_CASES[name], bs, spare=2, seed=bs)
    d = s.device()
    run_tables(paged, d, bs)
    s.check(d)


@pytest.mark.parametrize("rows", [4096, 4097, 4099, 9000])
def test_tables_pad_rows(paged, rows):
    s = TableState([3, 50, 0], [1, 4000, 0], 16, rows=rows)
    d = s.device()
    run_tables(paged, d, 16)
    s.check(d)


@pytest.mark.parametrize("shift", [1, 2])
def test_tables_odd_addresses(paged, shift):
    s = TableState([3, 50, 0], [1, 6000, 2], 16)
    d = s.device()
    for k in ("positions", "slots"):
        d[k] = ints([99] * (s.rows + shift))[shift:]
    wide = torch.full((3, s.columns + 5), 77, dtype=torch.int32, device=DEV)
    wide[:, :s.columns] = d["table"]
    d["table"] = wide[:, :s.columns]
    run_tables(paged, d, 16)
    s.check(d)
    assert (wide[:, s.columns:] == 77).all()


def test_tables_in_place(paged):
    s = TableState([3, 50, 0, 16, 200], [1, 400, 2, -1, 1], 16, spare=1)
    d = s.device()
    d["lens"], d["free_out"] = d["cached"], d["free_count"]
    run_tables(paged, d, 16)
    s.check(d)
    big = TableState([(i * 7) % 50 for i in range(6000)], [i % 4 - 1 for i in range(6000)], 32)
    d = big.device()
    d["lens"], d["free_out"] = d["cached"], d["free_count"]
    run_tables(paged, d, 32)
    big.check(d)


def failing():
    base = ([3, 50, 20], [1, 40, -1])
    yield "length", 1, base, lambda s: s.cached.__setitem__(0, -1)
    yield "columns", 1, base, lambda s: s.fresh.__setitem__(1, 1000)
    yield "huge", 1, base, lambda s: s.fresh.__setitem__(1, 2147483647)
    yield "rows", 2, base, lambda s: setattr(s, "rows", 40)
    yield "blocks", 4, ([3, 50, 0], [1, 40, 0]), lambda s: setattr(s, "count", s.count - 1)
    yield "count", 8, base, lambda s: setattr(s, "count", s.blocks + 1)
    yield "negative", 8, base, lambda s: setattr(s, "count", -1)
    yield "overfull", 8, base, lambda s: setattr(s, "count", s.blocks)
    yield "released", 16, base, lambda s: s.table[2].__setitem__(1, s.blocks)
    yield "handed", 16, ([3, 50, 0], [1, 40, 0]), lambda s: s.free.__setitem__(s.count - 1, -3)


@pytest.mark.parametrize("many", [0, 5000])
@pytest.mark.parametrize("name,bit,base,spoil", list(failing()), ids=[f[0] for f in failing()])
def test_tables_failures_change_nothing(paged, name, bit, base, spoil, many):
    s = TableState(list(base[0]) + [0] * many, list(base[1]) + [0] * many, 16, columns=6)
    spoil(s)
    d = s.device()
    run_tables(paged, d, 16)
    n = len(s.cached)
    assert d["status"].item() & bit
    assert d["table"].tolist() == s.table and d["lens"].tolist() == s.cached and d["free_out"].item() == s.count
    keep = max(0, min(s.count, s.blocks))
    assert d["free_list"].tolist()[:keep] == s.free[:keep]
    assert d["q_start"].tolist() == [0] * (n + 1)
    assert d["slots"].tolist() == [-1] * s.rows and d["positions"].tolist() == [0] * s.rows


# ---- append ---------------------------------------------------------------------


def make_cache(blocks, bs, heads, dim, dtype, layout, fill=0.0):
    shape = (blocks, bs, heads, dim) if layout == "token" else (blocks, heads, bs, dim)
    c = [torch.full(shape, fill, dtype=dtype, device=DEV) for _ in range(2)]
    return c if layout == "token" else [x.transpose(1, 2) for x in c]


@pytest.mark.parametrize("source,dtype", [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("rows,heads,dim,bs,layout", [(1, 8, 128, 16, "token"), (67, 3, 64, 32, "head"),
                                                     (1000, 20, 64, 128, "head"), (513, 1, 128, 64, "token")])
def test_append(paged, source, dtype, rows, heads, dim, bs, layout):
    g = torch.Generator(device=DEV).manual_seed(rows)
    blocks = rows // bs + 3
    kc, vc = make_cache(blocks, bs, heads, dim, dtype, layout, 7.0)
    both = torch.randn((rows, 2, heads, dim), device=DEV, generator=g).mul(40).to(source)
    both[0, 0, 0, :4] = torch.tensor([float("inf"), float("-inf"), float("nan"), -0.0], device=DEV).to(source)
    slots = torch.randperm(blocks * bs, device=DEV, generator=g)[:rows].int()
    if rows > 3:
        slots[2], slots[3] = -1, blocks * bs
    want = []
    for c, x in ((kc, both[:, 0]), (vc, both[:, 1])):
        w = c.clone()
        for i, s in enumerate(slots.tolist()):
            if 0 <= s < blocks * bs:
                w[s // bs, s % bs] = x[i].to(dtype)
        want.append(w)
    paged.append(both[:, 0], both[:, 1], kc, vc, slots)
    for c, w in zip((kc, vc), want):
        torch.testing.assert_close(c, w, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("source,dtype", [(F32, F32), (F32, BF16), (F16, F16)])
def test_append_odd_strides(paged, source, dtype):
    kc, vc = make_cache(4, 16, 2, 64, dtype, "token", 7.0)
    raw = torch.randn((9, 2 * 65 + 3), device=DEV).to(source)
    k = torch.as_strided(raw, (9, 2, 64), (133, 65, 1), 1)
    v = torch.as_strided(raw, (9, 2, 64), (133, 65, 1), 3)
    slots = ints([60, 3, 4, 5, -5, 17, 33, 1 << 30, 0])
    paged.append(k, v, kc, vc, slots)
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < 64:
            assert torch.equal(kc[s // 16, s % 16], k[i].to(dtype)) and torch.equal(vc[s // 16, s % 16], v[i].to(dtype))
    assert (kc == 7).sum() >= (64 - 7) * 2 * 64 - 8


def test_append_far_slots(paged):
    """Element offsets beyond 32 bits: 2.3 G elements of K."""
    blocks, bs, heads, dim = 18000, 128, 8, 128
    kc = torch.empty((blocks, bs, heads, dim), dtype=BF16, device=DEV)
    vc = torch.empty_like(kc)
    k = torch.randn((2, heads, dim), device=DEV)
    slots = [blocks * bs - 1, 17]
    paged.append(k, k * 2, kc, vc, ints(slots))
    for i, s in enumerate(slots):
        assert torch.equal(kc[s // bs, s % bs], k[i].to(BF16)) and torch.equal(vc[s // bs, s % bs], (k[i] * 2).to(BF16))
    # and the attention reads there: one key, so the output is its value row
    q = torch.randn((1, heads, dim), device=DEV).to(BF16)
    table = ints([[blocks - 1]])
    kc[blocks - 1], vc[blocks - 1] = 0, 3
    out = paged.attention(q, kc, vc, table, ints([bs]), ints([0, 1]), 1)
    assert torch.equal(out, torch.full_like(out, 3))


# ---- attention --------------------------------------------------------------------


class Step:
    """A step's inputs: requests of (fresh, cached), scattered blocks; what no row may see is NaN."""

    def __init__(self, requests, heads=4, kv=2, dim=64, bs=16, dtype=BF16, layout="token", pad=0, seed=0, junk=True,
                 qscale=1.5):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.bs, self.dtype, self.heads, self.kv, self.dim = bs, dtype, heads, kv, dim
        self.fresh, self.lens_h = [f for f, _ in requests], [max(0, f + c) for f, c in requests]
        used = [(n + bs - 1) // bs for n in self.lens_h]
        blocks = sum(used) + 2
        self.kc, self.vc = make_cache(blocks, bs, heads=kv, dim=dim, dtype=dtype, layout=layout,
                                      fill=float("nan") if junk else 0.0)
        ids = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
        columns = max(1, max(used)) + 1
        table = [[-1, blocks, 1 << 30][i % 3] for i in range(len(requests) * columns)]
        self.k, self.v = [], []
        for b, n in enumerate(self.lens_h):
            mine = [ids.pop() for _ in range(used[b])]
            table[b * columns:b * columns + used[b]] = mine
            k, v = (torch.randn((n, kv, dim), device=DEV, generator=g).to(dtype) for _ in range(2))
            for j, block in enumerate(mine):
                part = slice(j * bs, min(n, (j + 1) * bs))
                self.kc[block, :part.stop - part.start] = k[part]
                self.vc[block, :part.stop - part.start] = v[part]
            self.k.append(k)
            self.v.append(v)
        self.table = ints(table).view(len(requests), columns)
        start = [0] + list(itertools.accumulate(self.fresh))
        self.rows = start[-1] + pad
        self.start, self.lens, self.q_start = start, ints(self.lens_h), ints(start)
        self.q = (torch.randn((self.rows, heads, dim), device=DEV, generator=g) * qscale).to(dtype)
        if pad:
            self.q[start[-1]:] = float("nan")
        self.out = torch.full((self.rows, heads, dim), 5.0, dtype=dtype, device=DEV)

    def run(self, paged, max_fresh=None, **kw):
        return paged.attention(self.q, self.kc, self.vc, self.table, self.lens, self.q_start,
                               max_fresh or max(1, max(self.fresh)), out=self.out, **kw)

    def check(self, out, scale=None, drop=lambda b, j: False):
        """Against the definition in 64 bits.  The bound on an element counts, relative to a = sum p |v| / sum p:
        the rounding of the output (half a step of its value), of a 16-bit p (half a step of each term, so of a), the
        fp32 products and sums behind a score (dim + 2 roundings of sum |q k|, each to both the numerator and the
        denominator), the exponent's argument and result (2^-20 covers arguments up to 16 in size and the
        approximations of exp), and the fp32 sums over the n keys."""
        scale = self.dim ** -0.5 if scale is None else scale
        half = 0.0 if self.dtype is F32 else torch.finfo(self.dtype).eps / 2
        u = 2.0 ** -24
        group = self.heads // self.kv
        worst = 0.0
        for b, n in enumerate(self.lens_h):
            rows = slice(self.start[b], self.start[b + 1])
            f = rows.stop - rows.start
            if f == 0:
                continue
            seen = torch.arange(n, device=DEV)[None, :] <= (n - f + torch.arange(f, device=DEV))[:, None]
            for j in range((n + self.bs - 1) // self.bs):
                if drop(b, j):
                    seen[:, j * self.bs:(j + 1) * self.bs] = False
            for h in range(self.heads):
                q, k, v = self.q[rows, h].double(), self.k[b][:, h // group].double(), self.v[b][:, h // group].double()
                s = (q @ k.T * scale).masked_fill(~seen, -torch.inf)
                p = torch.softmax(s, -1).nan_to_num(0.0)  # a row without keys: zeros
                want, a = p @ v, p @ v.abs()
                size = (q.abs() @ k.abs().T * abs(scale)).masked_fill(~seen, 0.0)
                es = (self.dim + 2) * u * (size.amax(-1, keepdim=True) if n else 0.0)
                tol = torch.finfo(self.dtype).eps / 2 * want.abs() + a * (half + 2 * es + 2 * n * u + 2.0 ** -20) * 1.01
                got = out[rows, h].double()
                assert torch.isfinite(got).all(), (b, h)
                err = (got - want).abs()
                assert (err <= tol + 1e-30).all(), (b, h, float((err - tol).max()))
                worst = max(worst, float(err.max()))
        assert (out[self.start[-1]:] == 5).all()
        return worst


SHAPES = [(4, 2, 64), (16, 8, 128), (5, 5, 64), (3, 1, 128), (8, 1, 64), (34, 2, 64)]
MIXES = {
    "single": [(1, 0)],
    "steps": [(1, 0), (1, 1), (1, 14), (1, 15), (1, 16), (1, 127), (1, 128), (1, 300), (0, 50), (0, 0)],
    "few": [(2, 0), (5, 3), (3, 126), (8, 700), (1, 64), (7, 0)],
    "chunks": [(64, 0), (65, 63), (127, 1), (128, 128), (129, 300), (1, 77), (0, 9), (255, 2)],
    "empty_rows": [(5, -2), (3, -3), (1, -1), (40, -38), (130, -129), (4, 0)],
}


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
@pytest.mark.parametrize("mix", MIXES)
def test_attention(paged, mix, heads, kv, dim, dtype):
    i = SHAPES.index((heads, kv, dim))
    s = Step(MIXES[mix], heads, kv, dim, bs=[16, 32, 64, 128][i % 4], dtype=dtype, layout=["token", "head"][i % 2],
             pad=3, seed=i)
    s.check(s.run(paged))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("layout", ["token", "head"])
def test_attention_blocks(paged, bs, layout, dtype):
    s = Step([(1, 500), (77, 100), (1, 2 * bs - 1), (2, bs - 2), (1, bs)], 8, 4, 128, bs=bs, dtype=dtype, layout=layout)
    s.check(s.run(paged))
    s = Step([(1, 500), (2, bs - 2), (1, bs)], 8, 4, 64, bs=bs, dtype=dtype, layout=layout)
    s.check(s.run(paged))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("fresh,cached", [(1, 20000), (3, 9001), (300, 4000), (1024, 0)])
def test_attention_long(paged, fresh, cached, dtype):
    s = Step([(fresh, cached)], 4, 2, 128, bs=64, dtype=dtype)
    s.check(s.run(paged))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_many_requests(paged, dtype):
    s = Step([(1 + (i % 3 == 0), (i * 37) % 400) for i in range(300)], 4, 2, 64, bs=32, dtype=dtype)
    s.check(s.run(paged))
    s = Step([(i % 2, i % 5) for i in range(3000)], 2, 2, 64, bs=16, dtype=dtype)
    s.check(s.run(paged))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("mix", ["few", "chunks"])
def test_attention_is_right_whatever_max_fresh_says(paged, mix, dtype):
    for m in (1, 7, 5000):
        s = Step(MIXES[mix], 8, 4, 128, bs=32, dtype=dtype)
        s.check(s.run(paged, max_fresh=m))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("fresh", [1, 5, 200])
def test_attention_skips_bad_table_entries(paged, fresh, dtype):
    s = Step([(fresh, 500), (fresh, 90)], 4, 2, 128, bs=32, dtype=dtype)
    bad = {(0, 0): -1, (0, 4): 1 << 20, (0, 5): -2147483648, (1, 1): 2147483647, (1, 2): s.kc.shape[0]}
    for (b, j), v in bad.items():
        s.table[b, j] = v
    s.check(s.run(paged), drop=lambda b, j: (b, j) in bad)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("fresh", [1, 150])
def test_attention_without_any_good_block(paged, fresh, dtype):
    s = Step([(fresh, 100)], 4, 2, 64, bs=16, dtype=dtype)
    s.table[:] = -1
    out = s.run(paged)
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("fresh", [1, 40, 150])
def test_attention_keys_behind_the_table_are_not_seen(paged, fresh, dtype):
    s = Step([(fresh, 300)], 4, 2, 64, bs=16, dtype=dtype)
    s.table = s.table[:, :10].contiguous()
    s.check(s.run(paged), drop=lambda b, j: j >= 10)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_clamps_q_start(paged, dtype):
    s = Step([(3, 30), (4, 60)], 4, 2, 64, bs=16, dtype=dtype)
    s.q_start = ints([-5, 3, 900])
    # request 1 still ends at its length: only its last row count changes, so give it rows that fit
    s.lens = ints([33, 64])
    out = s.run(paged, max_fresh=8)
    assert torch.isfinite(out.float()).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("fresh", [1, 33, 200])
def test_attention_scales_and_extremes(paged, fresh, dtype):
    """Scores of hundreds, of one sign, all equal; a scale of zero and a negative one."""
    for scale, qscale in ((3.0, 4.0), (0.0, 1.0), (-0.2, 1.0)):
        s = Step([(fresh, 200)], 4, 2, 128, bs=64, dtype=dtype, qscale=qscale)
        out = s.run(paged, scale=scale)
        assert torch.isfinite(out.float()).all()
        if scale != 3.0:
            s.check(out, scale=scale)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("fresh", [1, 40])
def test_attention_nan_query_stays_in_its_row(paged, fresh, dtype):
    s = Step([(fresh, 100), (fresh, 30)], 4, 2, 64, bs=16, dtype=dtype)
    s.q[0, 1] = float("nan")
    out = s.run(paged).clone()
    assert torch.isnan(out[0, 1]).all()
    out[0, 1] = 0
    assert torch.isfinite(out.float()).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("fresh", [1, 20, 300])
def test_attention_strided_rows(paged, fresh, dtype):
    """q as a slice of a fused projection, out as a slice of a wider buffer."""
    s = Step([(fresh, 70), (2, 5)], 4, 2, 64, bs=16, dtype=dtype)
    wide = torch.full((s.rows, 4 * 64 + 128), float("nan"), dtype=dtype, device=DEV)
    wide[:, 64:64 + 256] = s.q.view(s.rows, 256)
    s.q = wide[:, 64:64 + 256].view(s.rows, 4, 64)
    room = torch.full((4, s.rows, 72), 5.0, dtype=dtype, device=DEV)
    s.out = room[:, :, :64].transpose(0, 1)
    s.check(s.run(paged))
    assert (room[:, :, 64:] == 5).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("mix", ["steps", "chunks"])
def test_attention_is_deterministic(paged, mix, dtype):
    s = Step(MIXES[mix] * 3, 8, 4, 128, bs=16, dtype=dtype)
    a = s.run(paged).clone()
    for _ in range(5):
        assert torch.equal(a, s.run(paged))


def test_attention_precision_f32(paged):
    """Normwise error of fp32 calls: a few fp32 roundings, not a 16-bit product."""
    for requests in ([(1, 3000)] * 4, [(300, 500)]):
        s = Step(requests, 8, 4, 128, bs=64, dtype=F32)
        out = s.run(paged).double()
        err = norm = 0.0
        for b, n in enumerate(s.lens_h):
            f = s.fresh[b]
            mask = torch.arange(n, device=DEV)[None, :] > (n - f + torch.arange(f, device=DEV))[:, None]
            for h in range(8):
                w = (s.q[s.start[b]:s.start[b + 1], h].double() @ s.k[b][:, h // 2].double().T * 128 ** -0.5)
                want = w.masked_fill(mask, -torch.inf).softmax(-1) @ s.v[b][:, h // 2].double()
                err += float((out[s.start[b]:s.start[b + 1], h] - want).square().sum())
                norm += float(want.square().sum())
        assert (err / norm) ** 0.5 < 1e-6


# ---- the operators together ----------------------------------------------------------


class Server:
    """Requests that come, grow and go over steps of tables, append and attention; every row is checked against
    dense attention over the request's history in 64 bits."""

    def __init__(self, paged, dtype, heads, kv, dim, bs, blocks, rows, batch, seed):
        self.paged, self.dtype, self.heads, self.kv, self.dim, self.bs, self.batch = paged, dtype, heads, kv, dim, bs, batch
        self.kc, self.vc = make_cache(blocks, bs, kv, dim, dtype, "head", float("nan"))
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.rows = rows
        self.lens, self.fresh = ints([0] * batch), ints([0] * batch)
        self.table = torch.full((batch, blocks), -1, dtype=torch.int32, device=DEV)
        self.free = torch.randperm(blocks, generator=self.g, device=DEV).int()
        self.count, self.status = ints([blocks]), ints([0])
        self.q_start = ints([0] * (batch + 1))
        self.positions, self.slots = ints([0] * rows), ints([0] * rows)
        self.qkv = torch.zeros((rows, (heads + 2 * kv), dim), device=DEV, dtype=dtype)
        self.out = torch.zeros((rows, heads, dim), device=DEV, dtype=dtype)
        self.history = [[] for _ in range(batch)]
        self.workspace = torch.empty(paged.workspace_bytes(dim), dtype=torch.uint8, device=DEV)

    def enqueue(self, max_fresh):
        p, h, kv = self.paged, self.heads, self.kv
        p.tables(self.lens, self.fresh, self.table, self.free, self.count, self.bs, lens=self.lens,
                 q_start=self.q_start, positions=self.positions, slots=self.slots, status=self.status)
        p.append(self.qkv[:, h:h + kv], self.qkv[:, h + kv:], self.kc, self.vc, self.slots)
        p.attention(self.qkv[:, :h], self.kc, self.vc, self.table, self.lens, self.q_start, max_fresh, out=self.out,
                    workspace=self.workspace)

    def fill(self, fresh):
        self.fresh.copy_(ints(fresh))
        self.qkv.copy_(torch.randn(self.qkv.shape, device=DEV, generator=self.g).to(self.dtype))

    def check(self, fresh):
        assert self.status.item() == 0
        half = 0.0 if self.dtype is F32 else torch.finfo(self.dtype).eps / 2
        t = 0
        for b, f in enumerate(fresh):
            if f < 0:
                self.history[b] = []
            for _ in range(max(f, 0)):
                self.history[b].append((self.qkv[t, self.heads:self.heads + self.kv].double(),
                                        self.qkv[t, self.heads + self.kv:].double()))
                assert self.positions[t].item() == len(self.history[b]) - 1
                k, v = (torch.stack(x) for x in zip(*self.history[b]))
                q = self.qkv[t, :self.heads].double().view(self.kv, -1, self.dim)
                s = torch.einsum("hgd,khd->hgk", q, k) * self.dim ** -0.5
                w = s.softmax(-1)
                want = torch.einsum("hgk,khd->hgd", w, v).reshape(self.heads, self.dim)
                size = torch.einsum("hgk,khd->hgd", w, v.abs()).reshape(self.heads, self.dim)
                tol = torch.finfo(self.dtype).eps / 2 * want.abs() + size * (half + 1e-4)
                assert ((self.out[t].double() - want).abs() <= tol).all(), (b, t)
                t += 1


STEPS = [[3, 0, 20, 1, 0], [1, 130, 1, 1, 0], [1, 1, -1, 1, 7], [-1, 1, 0, 1, 1], [40, 1, 33, -1, 1], [1, 1, 1, 2, 1],
         [-1, -1, -1, -1, -1], [17, 0, 0, 0, 1]]


@pytest.mark.parametrize("dtype,heads,kv,dim,bs", [(F32, 4, 2, 128, 16), (BF16, 6, 2, 64, 32), (F16, 4, 4, 128, 64)])
def test_steps_of_a_server(paged, dtype, heads, kv, dim, bs):
    s = Server(paged, dtype, heads, kv, dim, bs, blocks=40, rows=160, batch=5, seed=1)
    for fresh in STEPS:
        s.fill(fresh)
        s.enqueue(max(1, max(fresh)))
        s.check(fresh)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_steps_replayed_from_graphs(paged, dtype):
    """Two servers' steps captured into graphs (one bound of fresh rows for all steps), replayed in turn on two
    streams."""
    servers = [Server(paged, dtype, 4, 2, 64, 16, blocks=40, rows=160, batch=5, seed=i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in servers]
    graphs = []
    for s in servers:
        s.fill([0] * 5)
        s.enqueue(160)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.enqueue(160)
        graphs.append(g)
    for fresh in STEPS:
        for s in servers:
            s.fill(fresh)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for s in servers:
            s.check(fresh)


def test_side_stream_is_used(paged):
    """A call enqueues on the current stream: its inputs written earlier on that stream are seen."""
    s = Step([(1, 3000)] * 8, 8, 4, 128, bs=64, dtype=BF16)
    q = s.q.clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        s.q.zero_()
        torch.cuda._sleep(20_000_000)
        s.q.copy_(q)
        out = s.run(paged)
    side.synchronize()
    s.check(out)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("fresh", [1, 40, 200])
@pytest.mark.parametrize("what", ["k", "v"])
def test_attention_nan_key_reaches_every_row_that_sees_it(paged, fresh, dtype, what):
    """A NaN in one cached key or value row, at every offset within a few blocks of keys."""
    for j in range(64, 64 + 9):
        s = Step([(fresh, 300)], 4, 2, 64, bs=16, dtype=dtype)
        cache = s.kc if what == "k" else s.vc
        cache[s.table[0, j // 16].item(), j % 16, 1, 5] = float("nan")
        out = s.run(paged)
        assert torch.isfinite(out[:, :2].float()).all()
        assert torch.isnan(out[:, 2:, 5 if what == "v" else slice(None)]).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv,dim,bs", [(16, 8, 128, 64), (12, 12, 64, 128), (6, 2, 128, 128), (20, 20, 64, 16)])
def test_attention_many_units_per_cta(paged, heads, kv, dim, bs, dtype):
    """Enough work that every ring of the kernels goes round several times within an item and across items."""
    s = Step([(700, 2900), (1, 4100), (513, 1), (90, 6000), (255, 3333)], heads, kv, dim, bs=bs, dtype=dtype)
    s.check(s.run(paged))


# Row maps longer than one launch fills: a second grid finds each row's request.
LONG_MAPS = {
    "one": ([3], [16385]),
    "few": ([3, 50, 0, 700], [9000, 1, 0, 11000]),
    "steps": ([(11 * i) % 70 for i in range(8192)], [(i % 5) + 1 if i % 7 else 0 for i in range(8192)]),
    "ones": ([i % 33 for i in range(8192)], [1] * 4096 + [4] * 4096),
    "gaps": ([i % 20 for i in range(8000)],
             [17000] + [0] * 3000 + [7] * 100 + [-1] * 3000 + [900, 0, 1] + [0] * 1800 + [5] * 96),
}


@pytest.mark.parametrize("pad", [0, 1, 2, 3, 1500])
@pytest.mark.parametrize("name", LONG_MAPS)
def test_tables_long_maps(paged, name, pad):
    cached, fresh = LONG_MAPS[name]
    s = TableState(cached, fresh, 64, rows=sum(max(f, 0) for f in fresh) + pad, seed=pad)
    d = s.device()
    run_tables(paged, d, 64)
    s.check(d)


@pytest.mark.parametrize("rows", [16383, 16384, 16385])
def test_tables_long_map_edges(paged, rows):
    s = TableState([3, 50, 0], [1, 9000, 2], 16, rows=rows)
    d = s.device()
    run_tables(paged, d, 16)
    s.check(d)


@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("which", ["positions", "slots"])
def test_tables_long_map_odd_addresses(paged, which, shift):
    s = TableState([3, 50, 0], [1, 20000, 2], 16)
    d = s.device()
    whole = ints([99] * (s.rows + shift + 1))
    d[which] = whole[shift:shift + s.rows]
    run_tables(paged, d, 16)
    s.check(d)
    assert (whole[:shift] == 99).all() and whole[-1].item() == 99


@pytest.mark.parametrize("name,bit,base,spoil", [f for f in failing() if f[0] in ("length", "blocks", "released")],
                         ids=["length", "blocks", "released"])
def test_tables_long_map_failures(paged, name, bit, base, spoil):
    s = TableState(list(base[0]), list(base[1]), 16, columns=6, rows=20001)
    spoil(s)
    d = s.device()
    run_tables(paged, d, 16)
    assert d["status"].item() & bit
    assert d["table"].tolist() == s.table and d["lens"].tolist() == s.cached and d["free_out"].item() == s.count
    assert d["slots"].tolist() == [-1] * s.rows and d["positions"].tolist() == [0] * s.rows


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("max_fresh", [1, 32768])
def test_attention_without_measure_is_not_begun(paged, max_fresh, dtype):
    """Lengths of 2^30 for 32768 rows: in units of 256 rows by 64 keys, the largest, 2^7 2^24 128 = 2^38 of them, 3.5
    times the 2^29 for each of 148 CTAs."""
    rows, heads, dim, bs = 32768, 128, 128, 128
    cache = torch.zeros(2, bs, heads, dim, dtype=dtype, device=DEV)
    q = torch.zeros(1, heads, dim, dtype=dtype, device=DEV).expand(rows, heads, dim)
    out = torch.full((rows, heads, dim), 3.0, dtype=dtype, device=DEV)
    table = torch.full((1, 2 ** 30 // bs), -1, dtype=torch.int32, device=DEV)
    paged.attention(q, cache, cache, table, ints([2 ** 30]), ints([0, rows]), max_fresh, out=out)
    assert (out == 3).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_items_of_seconds(paged, dtype):
    """Items that take their CTA longer (3 and 4 s) than a wait for a unit may; their keys are one block, repeated."""
    heads, dim, bs = 148, 128, 128
    keys, fresh = (2 ** 26, 128) if dtype == F32 else (2 ** 28, 256)
    k = torch.zeros(1, bs, heads, dim, dtype=dtype, device=DEV)
    v = torch.zeros(1, bs, heads, dim, dtype=dtype, device=DEV)
    q = torch.ones(fresh, heads, dim, dtype=dtype, device=DEV)
    table = torch.zeros(1, keys // bs, dtype=torch.int32, device=DEV)
    out = paged.attention(q, k, v, table, ints([keys]), ints([0, fresh]), fresh)
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("fresh,dim,split", [(1, 128, False), (8, 64, False), (300, 128, False), (260, 64, False), (300, 128, True)])
@pytest.mark.parametrize("lift", [False, True])
def test_attention_long_sums(paged, fresh, dim, split, lift, dtype):
    """The mean of values that are all 1, over 2^19 + 77 keys, is 1, whether an item lies in one CTA or in many, and
    with the largest scores at the end (every sum before is scaled) or anywhere.

    Half a step of the type for the weights, which the products take rounded while their sum is not, and half a step
    for the output.  The sums: a step of 2^-23 of the sum for each 16 keys of at most 2^14 at a stretch (2^10 2^-23),
    2^-24 for each of the up to 2^5 stretches, and for a row's sum of weights the same for each 64 keys of a stretch;
    with 16 keys at a time, 2^15 sums to the nearest, whose errors of 2^-24 have either sign: 2^-24 2^7.5 and ten
    times that."""
    n, bs, requests = 2 ** 19 + 77, 128, 2 if split else 300
    g = torch.Generator(device=DEV).manual_seed(fresh + dim)
    blocks = (n + bs - 1) // bs
    k = torch.randn(blocks, bs, 1, dim, generator=g, device=DEV)
    q = torch.randn(fresh * requests, 1, dim, generator=g, device=DEV)
    if lift:
        q[:, :, 0] = 4.0
        k[-1, :, :, 0] = 12.0 * dim ** 0.5 / 8
    v = torch.ones(blocks, bs, 1, dim, dtype=dtype, device=DEV)
    table = torch.arange(blocks, dtype=torch.int32, device=DEV).expand(requests, blocks).contiguous()
    out = paged.attention(q.to(dtype), k.to(dtype), v, table, ints([n] * requests),
                          ints([fresh * b for b in range(requests + 1)]), fresh)
    assert (out.double() - 1).abs().max() <= torch.finfo(dtype).eps + 2 ** -13 + 2 ** -18


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("fresh", [1, 7, 200])
@pytest.mark.parametrize("what", ["heads", "tokens", "blocks", "rows", "query heads"])
def test_attention_reads_repeated_dimensions(paged, what, fresh, dtype):
    """Strides of 0 (expanded tensors) give what their copies give; within an allowance for another kernel's order."""
    g = torch.Generator(device=DEV).manual_seed(fresh)
    r = lambda *shape: torch.randn(*shape, generator=g, device=DEV).to(dtype)
    k, v, q = r(12, 32, 4, 64), r(12, 32, 4, 64), r(2 * fresh, 8, 64)
    if what == "heads":
        k, v = k[:, :, :1].expand(12, 32, 4, 64), v[:, :, 1:2].expand(12, 32, 4, 64)
    elif what == "tokens":
        k, v = k[:, :1].expand(12, 32, 4, 64), v[:, 5:6].expand(12, 32, 4, 64)
    elif what == "blocks":
        k, v = k[:1].expand(12, 32, 4, 64), v[3:4].expand(12, 32, 4, 64)
    elif what == "rows":
        q = q[:1].expand(2 * fresh, 8, 64)
    else:
        q = q[:, :1].expand(2 * fresh, 8, 64)
    table = ints([[0, 1, 2, 3, 4, 5, 6], [7, 8, 9, 10, 11, 0, 1]])
    rest = (table, ints([210, 201]), ints([0, fresh, 2 * fresh]), fresh)
    got = paged.attention(q, k, v, *rest).double()
    want = paged.attention(q.contiguous(), k.contiguous(), v.contiguous(), *rest).double()
    # both round weights and output to the type (half a step each); sums of 210 terms in fp32 otherwise
    top = v.double().abs().max()
    assert (got - want).abs().max() <= top * (2 * torch.finfo(dtype).eps + 210 * 2 ** -24)


def test_threads_with_their_own_streams(paged):
    """Four threads at once, each with its stream, type and shape, give what each gives alone."""
    import threading
    steps = [Step([(1, 500)] * 40, 16, 8, 128, bs=64, dtype=BF16, seed=1), Step(MIXES["chunks"], dtype=F32, seed=2),
             Step(MIXES["chunks"], 16, 8, 128, bs=128, dtype=F16, seed=3), Step(MIXES["few"], dtype=F32, seed=4)]
    alone = [s.run(paged).clone() for s in steps]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(50):
                    out = torch.empty_like(steps[i].q)
                    paged.attention(steps[i].q, steps[i].kc, steps[i].vc, steps[i].table, steps[i].lens,
                                    steps[i].q_start, max(steps[i].fresh), out=out)
                    if not torch.equal(out[:steps[i].start[-1]], alone[i][:steps[i].start[-1]]):
                        failed.append(i)
                try:
                    paged.attention(steps[i].q, steps[i].kc, steps[i].vc, steps[i].table, steps[i].lens,
                                    steps[i].q_start, 0)
                except ValueError as e:  # each thread has its own message
                    if "max_fresh" not in str(e):
                        failed.append(str(e))
        except Exception as e:  # noqa: BLE001
            failed.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
