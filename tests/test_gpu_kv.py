"""The 4-bit key/value cache on the GPU, against the plain 64-bit restatement in _kv_ref.py: pages and rows bit for bit, attention within
bounds derived there."""
import numpy as np
import pytest

import _kv_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def stream(torch):
    return torch.cuda.current_stream().cuda_stream


def as_type(torch, x, kind):
    """The tensor of fp64 values x in a type, and the values it then holds."""
    t = torch.from_numpy(np.ascontiguousarray(x)).to(torch.float32)
    t = t.to(torch.bfloat16 if kind == "bf16" else torch.float32)
    return t.cuda(), t.double().numpy()


def kv_type(kind):
    import zvdb_amd as zv
    return zv.KV_BF16 if kind == "bf16" else zv.KV_F32


# ---- plan -------------------------------------------------------------------------------------------------------------------------

def run_plan(torch, lengths, new, ring, cursor, tables, page, pages, slot_cap):
    import zvdb_amd as zv
    lay = zv.KVLayout(head_dim=64, kv_heads=1, page_size=page, pages=pages)
    n = len(lengths)
    i32 = lambda x: torch.tensor(np.asarray(x, dtype=np.uint32).view(np.int32), device="cuda")
    L, N, R, T = i32(lengths), i32(new), i32(ring), i32(tables)
    C = torch.tensor(np.asarray(cursor, np.int64), device="cuda")
    starts = torch.full((n + 1 + 3,), -7, dtype=torch.int32, device="cuda")
    slots = torch.full((slot_cap + 3,), -7, dtype=torch.int64, device="cuda")
    outl = torch.full((n + 3,), -7, dtype=torch.int32, device="cuda")
    outc, status = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.full((4,), -7, dtype=torch.int32, device="cuda")
    lay.plan_dev(L.data_ptr(), N.data_ptr(), n, R.data_ptr(), len(ring), C.data_ptr(), T.data_ptr(), tables.shape[1], starts.data_ptr(), slots.data_ptr(),
                 slot_cap, outl.data_ptr(), outc.data_ptr(), status.data_ptr(), stream(torch))
    torch.cuda.synchronize()
    h = lambda t: t.cpu().numpy()
    assert (h(starts)[n + 1:] == -7).all() and (h(slots)[slot_cap:] == -7).all() and (h(outl)[n:] == -7).all()
    return h(status), h(starts)[:n + 1], h(slots)[:slot_cap], h(outl)[:n], h(outc), h(T).view(np.uint32)


def check_plan(torch, lengths, new, ring, cursor, tables, page, pages, slot_cap):
    got = run_plan(torch, lengths, new, ring, cursor, tables, page, pages, slot_cap)
    code, starts, slots, outl, outc, tab, need, total = ref.plan(lengths, new, ring, cursor, tables, page, pages, slot_cap)
    assert got[0].tolist() == [code, min(need, 2**31 - 1), min(total, 2**31 - 1), 0]
    assert np.array_equal(got[1], starts) and np.array_equal(got[2], slots)
    assert np.array_equal(got[3].astype(np.int64) & 0xFFFFFFFF, np.asarray(outl)) and np.array_equal(got[4], np.asarray(outc))
    assert np.array_equal(got[5], tab)
    return code


def plan_case(rng, n, top_len, top_new, page, extra=0):
    lengths = rng.integers(0, top_len + 1, n)
    new = rng.integers(0, top_new + 1, n)
    held = int(sum(-(-c // page) for c in lengths))
    pages = held + int(sum(-(-(c + a) // page) for c, a in zip(lengths, new))) + 5
    order = rng.permutation(pages)
    stride = int(max([1] + [-(-(c + a) // page) for c, a in zip(lengths, new)])) + extra
    tables = np.full((n, stride), 0xFFFFFFFF, np.uint32)
    at = 0
    for i, c in enumerate(lengths):
        m = -(-int(c) // page)
        tables[i, :m] = order[at:at + m]
        at += m
    return lengths, new, order.astype(np.uint32), [held, pages], tables, pages


@pytest.mark.parametrize("n,top_len,top_new,page", [(1, 0, 1, 16), (1, 40, 1, 16), (3, 50, 0, 16), (64, 500, 1, 16), (65, 100, 70, 32), (300, 90, 33, 64), (1025, 40, 9, 16),
                                                    (2500, 300, 3, 256), (16384, 20, 2, 16), (7, 10, 4000, 128)])
def test_plan(torch, n, top_len, top_new, page):
    rng = np.random.default_rng(n * 7 + page)
    lengths, new, ring, cursor, tables, pages = plan_case(rng, n, top_len, top_new, page, extra=n % 3)
    total = int(new.sum())
    for cap in {total, total + 1, 2 * total + 37}:
        assert check_plan(torch, lengths, new, ring, cursor, tables, page, pages, cap) == 0


def test_plan_of_no_request(torch):
    assert check_plan(torch, [], [], np.arange(4, dtype=np.uint32), [1, 3], np.zeros((0, 1), np.uint32), 16, 4, 5) == 0


def test_plan_wraps_round_the_ring(torch):
    rng = np.random.default_rng(0)
    ring = rng.permutation(11).astype(np.uint32)
    tables = np.full((4, 3), 0xFFFFFFFF, np.uint32)
    for taken in (0, 5, 10, 11, 2**33 + 9):
        assert check_plan(torch, [0, 0, 0, 0], [17, 33, 1, 40], ring, [taken, taken + 11], tables, 16, 11, 91) == 0


@pytest.mark.parametrize("why", ["pages", "given behind taken", "table", "too long", "slots"])
def test_plan_is_all_or_nothing(torch, why):
    ring, cursor, stride, cap = np.arange(20, dtype=np.uint32), [3, 9], 4, 100
    lengths, new = [16, 5, 0], [16, 20, 33]  # 1 + 1 + 3 pages
    if why == "pages":
        cursor = [5, 9]
    elif why == "given behind taken":
        cursor = [9, 3]
    elif why == "table":
        stride = 2
    elif why == "too long":
        lengths[1], new[1] = 2**31 - 2, 2
    else:
        cap = 68
    tables = np.arange(3 * stride, dtype=np.uint32).reshape(3, stride)
    want = {"pages": 1, "given behind taken": 1, "table": 2, "too long": 2, "slots": 3}[why]
    assert check_plan(torch, lengths, new, ring, cursor, tables, 16, 20, cap) == want


def test_plan_of_entries_that_are_no_page(torch):
    """A partly filled page that is none, and a ring entry that is none: the tokens there get no slot."""
    tables = np.array([[7, 99, 0, 0], [1, 2, 0, 0]], np.uint32)
    assert check_plan(torch, [20, 16], [3, 20], np.array([3, 50, 4], np.uint32), [1, 4], tables, 16, 8, 30) == 0


# ---- append and read --------------------------------------------------------------------------------------------------------------

def special_rows(rng, n, heads, d):
    """Normal rows with the cases a block can be: zeros, ties, one large element, largest and smallest numbers, NaN, infinities."""
    x = rng.standard_normal((n, heads, d)) * np.exp2(rng.integers(-6, 7, (n, heads, 1)))
    x = x.reshape(n * heads, d)
    for r in range(len(x)):
        c, at = r % 13, 8 * (r % (d // 8))
        if c == 1:
            x[r] = 0
        elif c == 2:
            x[r] = rng.integers(-24, 25, d) * 0.25          # ties of the grid
        elif c == 3:
            x[r, at] = 3e38
        elif c == 4:
            x[r] = rng.standard_normal(d) * 2.0 ** -126
        elif c == 5:
            x[r, at] = np.nan
        elif c == 6:
            x[r, at + 7] = -np.inf
        elif c == 7:
            x[r] = 7.0 * np.sign(x[r])                       # 7/4 of a power of two: the scale doubles
        elif c == 8:
            x[r] = -0.0
        elif c == 9:
            x[r] = 6.999 * np.sign(x[r])
        elif c == 10:
            x[r] = rng.standard_normal(d) * 2.0 ** -140
    return x.reshape(n, heads, d)


@pytest.mark.parametrize("d,heads,page,n,kind", [(64, 1, 16, 1, "bf16"), (64, 3, 16, 37, "fp32"), (8, 2, 32, 21, "fp32"), (72, 2, 64, 33, "bf16"), (96, 4, 16, 50, "fp32"),
                                                 (128, 8, 128, 29, "bf16"), (128, 1, 16, 100, "fp32"), (136, 3, 16, 17, "bf16"), (256, 2, 256, 65, "bf16"),
                                                 (256, 1, 32, 40, "fp32"), (64, 5, 16, 70, "bf16"), (48, 7, 16, 19, "fp32"), (120, 5, 64, 31, "bf16"), (128, 6, 16, 40, "fp32"),
                                                 (128, 9, 32, 18, "bf16"), (200, 5, 16, 23, "bf16"), (256, 7, 64, 11, "fp32")])
def test_append_and_read_bit_for_bit(torch, d, heads, page, n, kind):
    import zvdb_amd as zv
    rng = np.random.default_rng(d + n)
    pages = -(-n // page) + 3
    lay = zv.KVLayout(head_dim=d, kv_heads=heads, page_size=page, pages=pages)
    fill = rng.integers(0, 256, pages * lay.page_bytes, dtype=np.uint8)
    cache = torch.from_numpy(fill.copy()).cuda()
    slots = rng.permutation(pages * page)[:n].astype(np.int64)
    slots[::9] = -1                      # no slot
    if n > 4:
        slots[4] = pages * page          # behind the cache
    row = heads * d
    ks, vs = row + 8, 2 * row + 16       # strides of their own, as in a fused projection's output
    with np.errstate(over="ignore"):
        (k, kx), (v, vx) = (as_type(torch, special_rows(rng, n, heads, d), kind) for _ in range(2))
    kbuf, vbuf = torch.zeros(n * ks, dtype=k.dtype, device="cuda"), torch.zeros(n * vs, dtype=k.dtype, device="cuda")
    kbuf.view(n, ks)[:, :row], vbuf.view(n, vs)[:, :row] = k.reshape(n, row), v.reshape(n, row)
    s_dev = torch.from_numpy(slots).cuda()
    lay.append_dev(cache.data_ptr(), kbuf.data_ptr(), ks, vbuf.data_ptr(), vs, kv_type(kind), n, s_dev.data_ptr(), stream(torch))
    want, vals = fill.copy(), [np.zeros((n, heads, d)) for _ in range(2)]
    for side, x in enumerate((kx, vx)):
        for h in range(heads):
            codes, scales, val = ref.encode_rows(x[:, h], d)
            for i, s in enumerate(slots):
                if 0 <= s < pages * page:
                    ref.put(want, d, heads, page, int(s), h, codes[i], scales[i], side == 1)
                    vals[side][i, h] = val[i]
    assert np.array_equal(cache.cpu().numpy(), want)
    for out in ("bf16", "fp32"):
        ok, ov = (torch.full((n + 1, heads, d), 5.0, dtype=torch.bfloat16 if out == "bf16" else torch.float32, device="cuda") for _ in range(2))
        lay.read_dev(cache.data_ptr(), s_dev.data_ptr(), n, ok.data_ptr(), ov.data_ptr(), kv_type(out), stream(torch))
        for o, x in zip((ok, ov), vals):
            assert np.array_equal(o.double().cpu().numpy()[:n], x, equal_nan=True) and (o[n] == 5.0).all()
        only = torch.empty_like(ov)      # one of the two
        lay.read_dev(cache.data_ptr(), s_dev.data_ptr(), n, 0, only.data_ptr(), kv_type(out), stream(torch))
        assert np.array_equal(only[:n].double().cpu().numpy(), vals[1], equal_nan=True)
        lay.read_dev(cache.data_ptr(), s_dev.data_ptr(), n, only.data_ptr(), 0, kv_type(out), stream(torch))
        assert np.array_equal(only[:n].double().cpu().numpy(), vals[0], equal_nan=True)


# ---- attention --------------------------------------------------------------------------------------------------------------------

class Memory:
    """A cache filled through append_dev, with the values that it then stands for; what no token wrote holds 0xFF (NaN scales)."""

    def __init__(self, torch, rng, lengths, d, heads, page, kind="fp32", stride=None, pages_more=2, spoil=None):
        import zvdb_amd as zv
        self.torch, self.lengths, self.d, self.heads, self.page = torch, list(lengths), d, heads, page
        need = [-(-x // page) for x in self.lengths]
        self.pages = sum(need) + pages_more
        self.lay = zv.KVLayout(head_dim=d, kv_heads=heads, page_size=page, pages=self.pages)
        self.cache = torch.full((self.pages * self.lay.page_bytes,), 255, dtype=torch.uint8, device="cuda")
        order = rng.permutation(self.pages)
        self.stride = stride or max([1] + need)
        self.tables = np.full((len(lengths), self.stride), 0xFFFFFFFF, np.uint32)
        at = 0
        slots = []
        for i, x in enumerate(self.lengths):
            self.tables[i, :need[i]] = order[at:at + need[i]]
            at += need[i]
            slots += [int(self.tables[i, p // page]) * page + p % page for p in range(x)]
        t = len(slots)
        self.first = np.concatenate(([0], np.cumsum(self.lengths))).astype(int)
        k, v = rng.standard_normal((2, t, heads, d)) * 1.5
        if spoil:
            spoil(self, k, v)
        (kt, kx), (vt, vx) = as_type(torch, k, kind), as_type(torch, v, kind)
        self.k, self.v = (np.stack([ref.encode_rows(x[:, h], d)[2] for h in range(heads)], 1) if t else np.zeros((0, heads, d)) for x in (kx, vx))
        s = torch.tensor(slots, dtype=torch.int64, device="cuda")
        if t:
            self.lay.append_dev(self.cache.data_ptr(), kt.data_ptr(), heads * d, vt.data_ptr(), heads * d, kv_type(kind), t, s.data_ptr(), stream(torch))

    def rows_of(self, i):
        return slice(self.first[i], self.first[i + 1])

    def i32(self, x):
        return self.torch.tensor(np.asarray(x, np.uint32).view(np.int32), device="cuda")


def attend(mem, q, new, group, kind, causal, scale, lengths=None, tables=None, max_new=None, max_length=None, rows=None, lse=True, ws=None, q_stride=None):
    torch = mem.torch
    heads, d = mem.heads * group, mem.d
    lengths = mem.lengths if lengths is None else lengths
    starts = np.concatenate(([0], np.cumsum(new))).astype(int)
    rows = starts[-1] if rows is None else rows
    max_new, max_length = max(new) if max_new is None else max_new, max(lengths) if max_length is None else max_length
    typ = kv_type(kind)
    out = torch.full((rows + 2, heads, d), 77.0, dtype=q.dtype, device="cuda")
    l = torch.full((rows + 2, heads), 77.0, device="cuda")
    size = mem.lay.attend_workspace(typ, heads, len(new), rows, max_new, max_length)
    if ws is None:
        ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    S, L, T = mem.i32(starts), mem.i32(lengths), mem.i32(mem.tables if tables is None else tables)
    mem.lay.attend_dev(mem.cache.data_ptr(), q.data_ptr(), q_stride or heads * d, typ, heads, len(new), S.data_ptr(), rows, max_new, L.data_ptr(), T.data_ptr(),
                       mem.stride, max_length, scale, causal, ws.data_ptr() if size else 0, size, out.data_ptr(), l.data_ptr() if lse else 0, stream(torch))
    torch.cuda.synchronize()
    return out.double().cpu().numpy(), l.double().cpu().numpy(), size


def check_rows(mem, got, lse, qx, rows, group, kind, scale, visible):
    """rows: (row, request); visible(row, request): the tokens of the request that the row sees, as a list of places."""
    for r, i in rows:
        see = visible(r, i)
        for h in range(mem.heads * group):
            kh, vh = mem.k[mem.rows_of(i)][see, h // group], mem.v[mem.rows_of(i)][see, h // group]
            with np.errstate(invalid="ignore"):
                o, l, bo, bl = ref.attend_row(qx[r, h], kh, vh, scale, kind)
            if np.isnan(kh).any():
                assert np.isnan(got[r, h]).all() and np.isnan(lse[r, h]), (r, h)
                continue
            bad = np.isnan(vh).any(0)
            assert np.array_equal(np.isnan(got[r, h]), bad), (r, h)
            assert (np.abs(got[r, h] - o)[~bad] <= bo[~bad]).all(), (r, h, np.abs(got[r, h] - o).max(), bo.max())
            assert lse[r, h] == l or abs(lse[r, h] - l) <= bl, (r, h, lse[r, h], l, bl)


def check_attend(torch, lengths, new, d, heads, group, page, kind, causal, seed=0, few=None, spoil=None, **kw):
    rng = np.random.default_rng(seed + d + sum(lengths))
    mem = Memory(torch, rng, lengths, d, heads, page, spoil=spoil)
    rows, qh = sum(new), heads * group
    q, qx = as_type(torch, 1.7 * rng.standard_normal((max(rows, 1), qh, d)), kind)
    scale = 1.0 / np.sqrt(d)
    got, lse, size = attend(mem, q, new, group, kind, causal, scale, **kw)
    owner = np.repeat(np.arange(len(new)), new)
    starts = np.concatenate(([0], np.cumsum(new))).astype(int)

    def visible(r, i):
        j = r - starts[i]
        return slice(0, max(0, lengths[i] - new[i] + j + 1) if causal else lengths[i])

    pick = range(rows) if few is None or rows <= few else sorted(set(rng.choice(rows, few, replace=False)) | {r for i, x in enumerate(new) if x for r in (starts[i], starts[i + 1] - 1)})
    check_rows(mem, got, lse, qx, [(r, owner[r]) for r in pick], group, kind, float(np.float32(scale)), visible)
    assert (got[rows:] == 77.0).all() and (lse[rows:] == 77.0).all()  # rows behind the last are left as they were
    return mem, q, got, lse, size


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("d,heads,group,page", [(64, 2, 1, 16), (64, 1, 7, 32), (80, 2, 3, 16), (128, 2, 4, 64), (128, 1, 16, 16), (96, 1, 33, 128), (256, 1, 5, 16), (200, 2, 2, 256)])
def test_single_tokens(torch, kind, d, heads, group, page):
    check_attend(torch, [1, 2, 15, 16, 17, 31, 32, 33, 100, 127, 129], [1] * 11, d, heads, group, page, kind, True)


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("d,heads,group,page", [(64, 1, 2, 16), (128, 2, 4, 16), (256, 1, 3, 64)])
def test_long_contexts_are_split_and_joined(torch, kind, d, heads, group, page):
    *_, size = check_attend(torch, [2500, 1, 1300], [1, 1, 1], d, heads, group, page, kind, True)
    assert size > 0  # (the call was split)


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("d,heads,group,page", [(64, 1, 2, 16), (40, 2, 1, 32), (128, 1, 3, 16), (104, 1, 2, 64), (256, 1, 2, 64), (248, 1, 1, 128)])
@pytest.mark.parametrize("bound,splits", [(2500, 5), (4096, 8), (4608, 9), (262_144, None)])
def test_every_number_of_splits(torch, kind, d, heads, group, page, bound, splits):
    # the host's bound says how many splits there are; the requests fill some of them, and a NaN key and a NaN value are in one each
    lengths, new = [2400, 0, 1, 2100, 1025], [1, 1, 1, 1, 1]

    def spoil(mem, k, v):
        k[mem.first[3] + 2099, 0, 1] = np.nan
        v[mem.first[4] + 1024, 0, d - 1] = np.inf

    with np.errstate(invalid="ignore"):
        *_, size = check_attend(torch, lengths, new, d, heads, group, page, kind, True, spoil=spoil, max_length=bound)
    part = len(new) * heads * group * (d + 4) * 4
    assert size == part * splits if splits else size > 9 * part


def test_the_largest_number_of_splits(torch):
    *_, size = check_attend(torch, [2100], [1], 64, 1, 2, 16, "bf16", True, max_length=262_144)
    assert size == 2 * 256 * (64 + 4) * 4


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,heads,group,page", [(64, 2, 2, 16), (128, 1, 4, 32), (72, 1, 5, 16), (256, 1, 2, 64)])
def test_prompts(torch, kind, causal, d, heads, group, page):
    # prompts over nothing, over a cache, one that leaves rows empty (more new tokens than tokens), none at all, a request without tokens
    check_attend(torch, [40, 300, 70, 0, 129, 0], [40, 77, 0, 3, 1, 0], d, heads, group, page, kind, causal, few=60)


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompts_of_many_rows(torch, kind, d):
    check_attend(torch, [700, 333], [513, 200], d, 1, 3, 16, kind, True, few=40)


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,new,d,heads,group", [
    ([900, 260, 0, 400, 311, 30], [300, 260, 0, 17, 290, 47], 64, 16, 2),             # rows that see nothing, requests of no row
    ([513, 700, 1500, 641, 600], [500, 641, 64, 641, 333], 128, 16, 2),
    ([5 * i % 97 + 60 for i in range(64)], [7 * i % 61 + 1 for i in range(64)], 64, 4, 3),
    ([5 * i % 97 + 60 for i in range(65)], [7 * i % 61 + 1 for i in range(65)], 64, 4, 3),
    ([900], [400], 104, 64, 2), ([700, 650], [300, 290], 128, 40, 2), ([700, 300], [300, 300], 56, 40, 2),  # two tiles to a wave
    ([400, 333], [300, 333], 256, 32, 2)])
def test_prompts_of_more_blocks_than_the_card_has_units(torch, kind, causal, lengths, new, d, heads, group):
    *_, got, lse, size = check_attend(torch, lengths, new, d, heads, group, 16, kind, causal, few=12)
    rows = sum(new)
    assert size == 0 and (got[:rows] != 77.0).all() and (lse[:rows] != 77.0).all()


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,new,d,heads,group", [
    ([1500, 40, 0, 900, 1211, 130], [100, 40, 3, 1, 61, 0], 64, 2, 3),
    ([1100, 600, 1300, 20], [90, 2, 130, 47], 128, 4, 2),
    ([1700, 310, 800], [40, 128, 3], 256, 4, 3)])
def test_prompts_in_splits_of_more_blocks_than_units(torch, kind, causal, lengths, new, d, heads, group):
    *_, got, lse, size = check_attend(torch, lengths, new, d, heads, group, 16, kind, causal, few=12)
    rows = sum(new)
    assert size > 0 and (got[:rows] != 77.0).all() and (lse[:rows] != 77.0).all()


def test_rows_without_tokens_get_zero_and_minus_infinity(torch):
    for new in ([5, 1], [90, 2]):
        mem, q, got, lse, _ = check_attend(torch, [2, 0], new, 64, 1, 1, 16, "bf16", True)
        assert (got[:new[0] - 2] == 0).all() and np.isneginf(lse[:new[0] - 2]).all()
        assert (got[new[0]:sum(new)] == 0).all() and np.isneginf(lse[new[0]:sum(new)]).all()


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("new", [1, 40])
def test_pages_that_are_none_hide_their_tokens(torch, kind, new):
    rng = np.random.default_rng(3)
    lengths, d, heads, group, page = [100, 48, 1400], 64, 2, 2, 16
    mem = Memory(torch, rng, lengths, d, heads, page)
    hide = {0: [0, 3, 6], 1: [0, 1, 2], 2: [1, 2, 40, 87]}
    tables = mem.tables.copy()
    for i, ps in hide.items():
        for n, p in enumerate(ps):
            tables[i, p] = (mem.pages, 0xFFFFFFFF, 0x80000000)[n % 3]
    q, qx = as_type(torch, rng.standard_normal((3 * new, heads * group, d)), kind)
    got, lse, _ = attend(mem, q, [new] * 3, group, kind, True, 0.25, tables=tables)

    def visible(r, i):
        return np.array([t for t in range(lengths[i] - new + r % new + 1) if t // page not in hide[i]], dtype=int)

    check_rows(mem, got, lse, qx, [(r, r // new) for r in range(3 * new)], group, kind, 0.25, visible)
    assert (got[new:2 * new] == 0).all() and np.isneginf(lse[new:2 * new]).all()


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("n,heads,long,new", [
    (512, 1, [4096 + 33, 8300], 1),                            # single tokens: 4,096 are what a wave knows the pages of at a time
    (130, 1, [1024 + 33, 2500], 128), (64, 2, [1024 + 1, 2100], 130)])  # prompts: 1,024
def test_long_contexts_that_are_not_split(torch, kind, d, page, n, heads, long, new):
    """Requests of many pages beside many short ones: too many blocks for splits, so that one goes through all of its request's pages.  Pages
    that are none, and NaN values, lie behind the first that it asks for."""
    group, rng = 2, np.random.default_rng(d + n)
    far = 4100 if new == 1 else 1030

    def spoil(mem, k, v):
        v[mem.first[1] + far + 20, 0, 7] = np.nan
        v[mem.first[1] + long[1] - 1, heads - 1, d - 1] = np.inf

    lengths = long + [i % 5 for i in range(n - 2)]
    with np.errstate(invalid="ignore"):
        mem = Memory(torch, rng, lengths, d, heads, page, spoil=spoil)
    hide = {0: [far // page], 1: [far // page - 1, far // page + 4]}
    tables = mem.tables.copy()
    for i, ps in hide.items():
        tables[i, ps] = mem.pages
    count = [new, new] + [min(x, 2) for x in lengths[2:]]
    starts = np.concatenate(([0], np.cumsum(count))).astype(int)
    q, qx = as_type(torch, rng.standard_normal((starts[-1], heads * group, d)), kind)
    got, lse, size = attend(mem, q, count, group, kind, True, 0.125, tables=tables)
    assert size == 0

    def visible(r, i):
        return np.array([t for t in range(lengths[i] - count[i] + r - starts[i] + 1) if t // page not in hide.get(i, [])], dtype=int)

    rows = [(0, 0), (new - 1, 0), (new, 1), (2 * new - 1, 1)] + [(starts[i], i) for i in (5, 6, n - 1) if count[i]]
    check_rows(mem, got, lse, qx, rows, group, kind, 0.125, visible)


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_nan_reaches_the_rows_that_see_it_and_no_others(torch, kind, d):
    def spoil(mem, k, v):
        v[30, 0, 33] = np.nan         # one block of one value
        v[61, 1, 0] = np.inf
        k[45, 1, d - 1] = -np.inf     # a key: everything of the rows that see it
    check_attend(torch, [70], [64], d, 2, 2, 16, kind, True, spoil=spoil)
    check_attend(torch, [70], [3], d, 2, 2, 16, kind, True, spoil=spoil)
    check_attend(torch, [50], [40], d, 1, 2, 16, kind, False, spoil=lambda mem, k, v: v.__setitem__((30, 0, 33), np.nan))


def loud_key(mem, k, request, token, head=slice(None)):
    """Queries of check_loud have 8 in element 0, where only this token's key is not 0: it scores hundreds above all others."""
    k[mem.first[request] + token, head, 0] = 1000.0


def check_loud(torch, lengths, new, d, heads, group, kind, causal, spoil, few=None, **kw):
    """As check_attend, with queries that meet loud_key."""
    rng = np.random.default_rng(d + sum(lengths))

    def all_of_it(mem, k, v):
        k[:, :, 0] = 0.0
        spoil(mem, k, v)

    with np.errstate(invalid="ignore"):
        mem = Memory(torch, rng, lengths, d, heads, 16, spoil=all_of_it)
    x = rng.standard_normal((sum(new), heads * group, d))
    x[:, :, 0] = 8.0
    q, qx = as_type(torch, x, kind)
    scale, starts = 1.0 / np.sqrt(d), np.concatenate(([0], np.cumsum(new))).astype(int)
    got, lse, size = attend(mem, q, new, group, kind, causal, scale, **kw)
    owner = np.repeat(np.arange(len(new)), new)
    pick = range(sum(new)) if few is None or sum(new) <= few else sorted(set(rng.choice(sum(new), few, replace=False)) | set(starts[:-1]) | set(starts[1:] - 1))
    check_rows(mem, got, lse, qx, [(r, owner[r]) for r in pick], group, kind, float(np.float32(scale)),
               lambda r, i: slice(0, lengths[i] - new[i] + r - starts[i] + 1 if causal else lengths[i]))
    return got, size


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,bound", [([1, 1, 1], 4096), ([1, 1, 1], 4608), ([60, 1, 33], 2500)])  # eight splits, nine, prompts
def test_a_nan_is_kept_where_its_split_weighs_nothing(torch, kind, d, new, bound):
    """One key outweighs every other split of its request by more than fp32 can hold; the NaN of a value lies in another one, before or
    behind it, and reaches the rows all the same: 0 NaN is NaN."""
    def spoil(mem, k, v):
        loud_key(mem, k, 0, 10), loud_key(mem, k, 1, 2040)
        v[mem.first[0] + 2300, 0, 3] = np.nan
        v[mem.first[1] + 5, 1, d - 1] = np.inf
        v[mem.first[1] + 700, 0, 0] = -np.inf

    got, size = check_loud(torch, [2400, 2100, 90], new, d, 2, 2, kind, True, spoil, few=8, max_length=bound)
    assert size > 0 and np.isnan(got[0]).any() and np.isnan(got[new[0]]).any()


def check_sizes(torch, lengths, new, d, heads, group, kind, causal, power=125, few=None, **kw):
    """Values of 2^power -- a block holds up to 6 x 2^125 -- against scores that differ by less than the slack of a running maximum: what
    a sum of exponentials times the largest comes to before it is divided does not fit fp32."""
    def spoil(mem, k, v):
        k[:] = 0.0
        for i, t in enumerate(lengths):
            k[mem.first[i] + t // 2:mem.first[i + 1], :, 0] = 4.0    # 4.5 more (6.5 as powers of two) in the second half
            k[mem.first[i] + t - 1:mem.first[i + 1], :, 0] = 3.0
        v[:, :, ::4] = np.abs(v[:, :, ::4]) * 2.0 ** power            # columns of one sign
        v[:, :, 1::4] *= 2.0 ** power                                 # and of both
        np.clip(v, -2.5e38, 2.5e38, out=v)

    rng = np.random.default_rng(d + sum(lengths))
    mem = Memory(torch, rng, lengths, d, heads, 16, spoil=spoil)
    x = rng.standard_normal((sum(new), heads * group, d))
    x[:, :, 0] = 4.5 * np.sqrt(d) / 4.0
    q, qx = as_type(torch, x, kind)
    scale, starts = 1.0 / np.sqrt(d), np.concatenate(([0], np.cumsum(new))).astype(int)
    got, lse, size = attend(mem, q, new, group, kind, causal, scale, **kw)
    owner = np.repeat(np.arange(len(new)), new)
    pick = range(sum(new)) if few is None or sum(new) <= few else sorted(set(rng.choice(sum(new), few, replace=False)) | set(starts[:-1]) | set(starts[1:] - 1))
    check_rows(mem, got, lse, qx, [(r, owner[r]) for r in pick], group, kind, float(np.float32(scale)),
               lambda r, i: slice(0, lengths[i] - new[i] + r - starts[i] + 1 if causal else lengths[i]))
    return mem, q, qx, size


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lengths,new,bound,split", [
    ([2, 33, 64, 100, 257, 1000], [1] * 6, 1000, False), ([2400, 700, 3], [1] * 3, 4096, True), ([2400, 700, 3], [1] * 3, 4608, True),  # single tokens
    ([300, 130], [40, 129], 300, None), ([2100, 900], [60, 70], 2100, True)])                                                          # prompts
def test_values_near_the_largest_stay_finite(torch, kind, d, lengths, new, bound, split):
    *_, size = check_sizes(torch, lengths, new, d, 2, 2, kind, True, few=8, max_length=bound)
    assert split is None or (size > 0) == split


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_small_values_keep_their_bits(torch, kind, d):
    for new in ([1, 1], [60, 70]):
        check_sizes(torch, [300, 2100], new, d, 2, 2, kind, True, power=-108, few=8)


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("length,new,heads", [(40, 1, 1), (2100, 1, 1), (40, 33, 2), (1500, 70, 2), (300, 280, 32)])
def test_rows_whose_scores_are_all_minus_infinity(torch, kind, d, length, new, heads):
    """Finite queries and keys whose products leave fp32 downwards: no token has a weight, as where none is seen."""
    def spoil(mem, k, v):
        k[:] = 0.0
        k[:, :, 5] = 6.0

    mem = Memory(torch, np.random.default_rng(d), [length], d, heads, 16, spoil=spoil)
    q = torch.zeros((new, 2 * heads, d), dtype=torch.bfloat16 if kind == "bf16" else torch.float32, device="cuda")
    q[:, :, 5] = -3e38
    got, lse, _ = attend(mem, q, [new], 2, kind, True, 0.125)
    assert (got[:new] == 0).all() and np.isneginf(lse[:new]).all()
    if new == 1:
        ids = np.tile(np.arange(length, dtype=np.uint64), (heads, 1, 1))
        got, lse = selected(mem, q, ids, None, 2, kind, 0.125)
        assert (got[:1] == 0).all() and np.isneginf(lse[:1]).all()


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("query,scale", [(3e38, 0.125), (4.0, 1e38)])  # a product, and a finite product's score, over all of fp32
@pytest.mark.parametrize("length,new,heads", [(40, 1, 1), (2100, 1, 1), (40, 33, 2), (1500, 70, 2), (300, 280, 32)])
def test_rows_with_a_score_over_all_of_fp32_are_nan(torch, kind, d, query, scale, length, new, heads):
    """The last token that the first row sees has such a score, all others 0; rows of request 1, whose keys are 0, have their means."""
    def spoil(mem, k, v):
        k[:] = 0.0
        k[length - new, :, 5] = 6.0

    mem = Memory(torch, np.random.default_rng(d), [length, 50], d, heads, 16, spoil=spoil)
    q = torch.zeros((new + 1, 2 * heads, d), dtype=torch.bfloat16 if kind == "bf16" else torch.float32, device="cuda")
    q[:, :, 5] = query
    got, lse, _ = attend(mem, q, [new, 1], 2, kind, True, scale)
    assert np.isnan(got[:new]).all() and np.isnan(lse[:new]).all()
    assert np.isfinite(got[new]).all() and np.abs(lse[new] - np.log(50)).max() < 1e-5
    if new == 1:
        ids = np.tile(np.arange(length, dtype=np.uint64), (heads, 2, 1))
        got, lse = selected(mem, q, ids, None, 2, kind, scale)
        assert np.isnan(got[0]).all() and np.isnan(lse[0]).all() and np.isfinite(got[1]).all()


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("d,heads", [(64, 16), (128, 16), (256, 32)])
def test_values_near_the_largest_in_whole_prompts(torch, kind, d, heads):
    *_, size = check_sizes(torch, [400, 700], [300, 290], d, heads, 2, kind, False, few=4)
    assert size == 0


def test_scores_of_any_size(torch):
    """Large scores, rows whose maximum moves late, all scores equal, all far below zero."""
    def spoil(mem, k, v):
        k[:] = 0
        k[10:, :, 0] = 8.0
        k[200:, :, 1] = -64.0
        k[290] = 24.0
    for kind in ("bf16", "fp32"):
        for new in (1, 80):
            check_attend(torch, [300], [new], 64, 1, 2, 16, kind, True, spoil=spoil)


def test_bounds_that_the_host_states(torch):
    """A longer request than max_length is seen up to it; tokens beyond a table row are not; rows behind max_new are left."""
    rng = np.random.default_rng(9)
    mem = Memory(torch, rng, [200, 90], 64, 1, 16)
    q, qx = as_type(torch, rng.standard_normal((6, 2, 64)), "fp32")
    got, lse, _ = attend(mem, q, [3, 3], 2, "fp32", True, 0.2, max_length=100)
    check_rows(mem, got, lse, qx, [(r, r // 3) for r in range(6)], 2, "fp32", float(np.float32(0.2)), lambda r, i: slice(0, 100 if i == 0 else 88 + r % 3))
    got, lse, _ = attend(mem, q, [3, 3], 2, "fp32", False, 0.2, max_new=2)
    check_rows(mem, got, lse, qx, [(r, r // 3) for r in (0, 1, 3, 4)], 2, "fp32", float(np.float32(0.2)), lambda r, i: slice(0, mem.lengths[i]))
    assert (got[[2, 5]] == 77.0).all()
    mem.stride = 13  # row 0: 13 pages of 16 = 208 tokens that the table can name; the request says more
    got, lse, _ = attend(mem, q, [3, 3], 2, "fp32", False, 0.2, lengths=[5000, 90], tables=mem.tables[:, :13])
    check_rows(mem, got, lse, qx, [(r, 1) for r in (3, 4, 5)], 2, "fp32", float(np.float32(0.2)), lambda r, i: slice(0, 90))


def test_starts_that_reach_behind_the_rows_stay_inside(torch):
    rng = np.random.default_rng(10)
    mem = Memory(torch, rng, [64, 64], 64, 1, 16)
    q, qx = as_type(torch, rng.standard_normal((4, 1, 64)), "bf16")
    got, lse, _ = attend(mem, q, [2, 40], 1, "bf16", False, 0.2, rows=4, max_new=40)
    check_rows(mem, got, lse, qx, [(r, r // 2) for r in range(4)], 1, "bf16", float(np.float32(0.2)), lambda r, i: slice(0, 64))
    assert (got[4:] == 77.0).all()


def test_strided_queries_and_no_lse(torch):
    rng = np.random.default_rng(11)
    mem = Memory(torch, rng, [77, 5], 64, 2, 16)
    wide, wx = as_type(torch, rng.standard_normal((5, 3 * 4 * 64 + 8)), "bf16")  # a fused projection's rows
    got, lse, _ = attend(mem, wide, [3, 2], 2, "bf16", True, 0.125, q_stride=wide.shape[1], lse=False)
    qx = wx[:, :256].reshape(5, 4, 64)
    assert (lse == 77.0).all()
    _, full, _ = attend(mem, wide, [3, 2], 2, "bf16", True, 0.125, q_stride=wide.shape[1])
    check_rows(mem, got, full, qx, [(0, 0), (1, 0), (2, 0), (3, 1), (4, 1)], 2, "bf16", 0.125, lambda r, i: slice(0, mem.lengths[i] - (3, 2)[i] + (r - 3 * i) + 1))


@pytest.mark.parametrize("new", [1, 65])
def test_the_same_inputs_give_the_same_bits(torch, new):
    rng = np.random.default_rng(12)
    mem = Memory(torch, rng, [1500, 900], 128, 2, 16)
    q, _ = as_type(torch, rng.standard_normal((2 * new, 8, 128)), "bf16")
    a = attend(mem, q, [new, new], 4, "bf16", True, 0.1)
    for _ in range(3):
        b = attend(mem, q, [new, new], 4, "bf16", True, 0.1)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_a_workspace_that_is_too_small_is_refused(torch):
    import zvdb_amd as zv
    rng = np.random.default_rng(13)
    mem = Memory(torch, rng, [1500], 64, 1, 16)
    q, _ = as_type(torch, rng.standard_normal((1, 1, 64)), "bf16")
    size = mem.lay.attend_workspace(zv.KV_BF16, 1, 1, 1, 1, 1500)
    ws, out, S, L, T = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.empty_like(q), mem.i32([0, 1]), mem.i32([1500]), mem.i32(mem.tables)
    for p, b in ((ws.data_ptr(), size - 1), (0, size), (ws.data_ptr() + 8, size)):
        with pytest.raises(zv.ZvdbError) as e:
            mem.lay.attend_dev(mem.cache.data_ptr(), q.data_ptr(), 64, zv.KV_BF16, 1, 1, S.data_ptr(), 1, 1, L.data_ptr(), T.data_ptr(), mem.stride, 1500, 0.1, True, p, b,
                               out.data_ptr(), 0, stream(torch))
        assert e.value.code == 1


def test_one_workspace_for_batches_of_every_size(torch):
    """The need does not grow with the batch: the largest answer over the sizes in use serves them all, the largest batch's alone does not."""
    import zvdb_amd as zv
    rng = np.random.default_rng(61)
    mem = Memory(torch, rng, [40 + 37 * (i % 31) for i in range(64)], 64, 8, 16)
    q, qx = as_type(torch, rng.standard_normal((64, 8, 64)), "bf16")
    sizes = {n: mem.lay.attend_workspace(zv.KV_BF16, 8, n, n, 1, 8192) for n in range(1, 65)}
    assert sizes[64] == 0 and max(sizes.values()) == max(sizes[n] for n in range(1, 64)) > 0
    ws = torch.full((max(sizes.values()),), 255, dtype=torch.uint8, device="cuda")
    lengths, tables, starts = mem.i32(mem.lengths), mem.i32(mem.tables), mem.i32(range(65))
    out, lse = torch.empty((64, 8, 64), dtype=torch.bfloat16, device="cuda"), torch.empty((64, 8), device="cuda")

    def call(n, have):
        mem.lay.attend_dev(mem.cache.data_ptr(), q.data_ptr(), 512, zv.KV_BF16, 8, n, starts.data_ptr(), n, 1, lengths.data_ptr(), tables.data_ptr(), mem.stride, 8192,
                           0.125, True, ws.data_ptr(), have, out.data_ptr(), lse.data_ptr(), stream(torch))
        torch.cuda.synchronize()

    for n in (64, 63, 48, 33, 16, 5, 1):
        out.fill_(77.0), lse.fill_(77.0)
        call(n, ws.numel())
        got, l = out.double().cpu().numpy(), lse.double().cpu().numpy()
        check_rows(mem, got, l, qx, [(r, r) for r in range(0, n, 7)], 1, "bf16", 0.125, lambda r, i: slice(0, mem.lengths[i]))
        assert (got[n:] == 77.0).all() and (got[:n] != 77.0).all()
    with pytest.raises(zv.ZvdbError) as e:
        call(16, sizes[64])
    assert e.value.code == 1


def test_host_memory_is_refused(torch):
    import zvdb_amd as zv
    lay = zv.KVLayout(head_dim=64, kv_heads=1, page_size=16, pages=1)
    for pin in (False, True):
        host = torch.zeros(1 << 16, dtype=torch.uint8)
        host = host.pin_memory() if pin else host
        dev = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
        at = (host.data_ptr() + 15) // 16 * 16
        with pytest.raises(zv.ZvdbError) as e:
            lay.read_dev(at, dev.data_ptr(), 1, dev.data_ptr(), 0, 0, stream(torch))
        assert e.value.code == 1


def test_a_cache_beyond_32_bits_of_bytes(torch):
    """Pages behind 4 GiB and behind 2^31 slots' worth of bytes: the same answers as in a small cache."""
    rng = np.random.default_rng(14)
    import zvdb_amd as zv
    mem = Memory(torch, rng, [300, 65], 128, 2, 16)
    big = zv.KVLayout(head_dim=128, kv_heads=2, page_size=16, pages=(10 << 30) // mem.lay.page_bytes)
    far = torch.empty(big.pages * big.page_bytes, dtype=torch.uint8, device="cuda")
    move = big.pages - mem.pages
    far[move * big.page_bytes:] = mem.cache
    q, _ = as_type(torch, rng.standard_normal((42, 4, 128)), "bf16")
    for new in ([1, 1], [40, 2]):
        want = attend(mem, q, new, 2, "bf16", True, 0.1)
        small = (mem.lay, mem.cache, mem.tables)
        mem.lay, mem.cache, mem.tables = big, far, np.where(mem.tables < mem.pages, mem.tables + move, mem.tables).astype(np.uint32)
        got = attend(mem, q, new, 2, "bf16", True, 0.1)
        mem.lay, mem.cache, mem.tables = small
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    slots = torch.tensor([move * 16 + 3, big.pages * 16 - 1], device="cuda")
    k = torch.randn(2, 2, 128, device="cuda")
    big.append_dev(far.data_ptr(), k.data_ptr(), 256, k.data_ptr(), 256, zv.KV_F32, 2, slots.data_ptr(), stream(torch))
    mem.lay.append_dev(mem.cache.data_ptr(), k.data_ptr(), 256, k.data_ptr(), 256, zv.KV_F32, 2, (slots - move * 16).data_ptr(), stream(torch))
    assert torch.equal(far[move * big.page_bytes:], mem.cache)
    a, b = torch.empty_like(k), torch.empty_like(k)
    big.read_dev(far.data_ptr(), slots.data_ptr(), 2, a.data_ptr(), b.data_ptr(), zv.KV_F32, stream(torch))
    assert torch.equal(a, b) and torch.isfinite(a).all()


# ---- attention over selected rows -------------------------------------------------------------------------------------------------

def selected(mem, q, ids, counts, group, kind, scale, lengths=None):
    torch = mem.torch
    heads, n, k = ids.shape
    qh = heads * group
    out = torch.full((n + 1, qh, mem.d), 77.0, dtype=q.dtype, device="cuda")
    lse = torch.full((n + 1, qh), 77.0, device="cuda")
    I = torch.tensor(ids.astype(np.uint64).view(np.int64), device="cuda")
    C = mem.i32(counts) if counts is not None else None
    L, T = mem.i32(mem.lengths if lengths is None else lengths), mem.i32(mem.tables)
    mem.lay.attend_selected_dev(mem.cache.data_ptr(), q.data_ptr(), qh * mem.d, kv_type(kind), qh, n, I.data_ptr(), C.data_ptr() if C is not None else 0, k,
                                L.data_ptr(), T.data_ptr(), mem.stride, scale, out.data_ptr(), lse.data_ptr(), stream(torch))
    torch.cuda.synchronize()
    assert (out[n] == 77.0).all() and (lse[n] == 77.0).all()
    return out.double().cpu().numpy(), lse.double().cpu().numpy()


def check_selected(mem, got, lse, qx, ids, counts, group, kind, scale, there=None):
    heads, n, k = ids.shape
    for i in range(n):
        for h in range(heads * group):
            m = k if counts is None else min(int(counts[h // group, i]), k)
            see = [int(t) for t in ids[h // group, i, :m] if int(t) < mem.lengths[i] and (there is None or there(i, int(t)))]
            kh, vh = mem.k[mem.rows_of(i)][see, h // group], mem.v[mem.rows_of(i)][see, h // group]
            with np.errstate(invalid="ignore"):
                o, l, bo, bl = ref.attend_row(qx[i, h], kh, vh, scale, kind)
            if np.isnan(kh).any():
                assert np.isnan(got[i, h]).all() and np.isnan(lse[i, h])
                continue
            bad = np.isnan(vh).any(0)
            assert np.array_equal(np.isnan(got[i, h]), bad), (i, h)
            assert (np.abs(got[i, h] - o)[~bad] <= bo[~bad]).all(), (i, h)
            assert lse[i, h] == l or abs(lse[i, h] - l) <= bl, (i, h, lse[i, h], l)


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("d,heads,group,page,k", [(64, 2, 1, 16, 10), (64, 1, 4, 32, 1), (96, 2, 3, 16, 33), (128, 2, 4, 64, 100), (128, 1, 20, 16, 129), (256, 1, 2, 16, 40),
                                                  (64, 1, 2, 16, 1100)])
def test_selected_rows(torch, kind, d, heads, group, page, k):
    rng = np.random.default_rng(d + k)
    lengths = [300, 1, 77, 1500 if k > 1000 else 40]
    mem = Memory(torch, rng, lengths, d, heads, page)
    n = len(lengths)
    ids = rng.integers(0, 1500, (heads, n, k)).astype(np.uint64)          # many are behind the request's tokens; some twice
    for h in range(heads):
        for i in range(n):
            ids[h, i, ::2] = rng.integers(0, lengths[i], len(ids[h, i, ::2]))
    ids[:, :, k // 2] = 2**64 - 1
    ids[:, 2, -1] = 2**32 + 5                                              # not token 5
    counts = rng.integers(0, k + 1, (heads, n))
    counts[0, 0], counts[-1, 1], counts[0, 2] = k, 0, k + 7                # more than k is k
    q, qx = as_type(torch, rng.standard_normal((n, heads * group, d)), kind)
    for c in (counts, None):
        got, lse = selected(mem, q, ids, c, group, kind, 0.3)
        check_selected(mem, got, lse, qx, ids, c, group, kind, float(np.float32(0.3)))


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("d,k", [(64, 2049), (128, 1024), (128, 1100), (256, 1025), (256, 2100)])
def test_long_lists_of_selected_rows(torch, kind, d, k):
    """More entries than are resolved at a time, some that are not there, a NaN behind the first 1,024."""
    rng = np.random.default_rng(d + k)
    lengths = [1500, 700]

    def spoil(mem, key, v):
        v[mem.first[0] + 1499, 0, 9] = np.nan

    mem = Memory(torch, rng, lengths, d, 2, 32, spoil=spoil)
    ids = np.stack([np.stack([rng.integers(0, x - 1, k) for x in lengths]) for _ in range(2)]).astype(np.uint64)
    ids[:, :, 5::11] = 2**64 - 1
    ids[:, 1, 7::13] = 700
    ids[0, 0, -1] = 1499
    counts = np.array([[k, k - 1], [k - 20, k]])
    q, qx = as_type(torch, rng.standard_normal((2, 4, d)), kind)
    got, lse = selected(mem, q, ids, counts, 2, kind, 0.3)
    assert np.isnan(got[0, 0, 9])
    check_selected(mem, got, lse, qx, ids, counts, 2, kind, float(np.float32(0.3)))


@pytest.mark.parametrize("d", [64, 128, 256])
def test_selected_rows_beyond_32_bits_of_bytes(torch, d):
    """Pages behind 4 GiB: the same answers as in a small cache."""
    import zvdb_amd as zv
    rng = np.random.default_rng(15)
    mem = Memory(torch, rng, [300, 65], d, 2, 16)
    big = zv.KVLayout(head_dim=d, kv_heads=2, page_size=16, pages=(10 << 30) // mem.lay.page_bytes)
    far = torch.empty(big.pages * big.page_bytes, dtype=torch.uint8, device="cuda")
    move = big.pages - mem.pages
    far[move * big.page_bytes:] = mem.cache
    ids = np.stack([np.stack([rng.permutation(300)[:60] for _ in range(2)]) for _ in range(2)]).astype(np.uint64)
    for kind in ("bf16", "fp32"):
        q, qx = as_type(torch, rng.standard_normal((2, 4, d)), kind)
        want = selected(mem, q, ids, None, 2, kind, 0.1)
        check_selected(mem, *want, qx, ids, None, 2, kind, float(np.float32(0.1)))
        small = (mem.lay, mem.cache, mem.tables)
        mem.lay, mem.cache, mem.tables = big, far, np.where(mem.tables < mem.pages, mem.tables + move, mem.tables).astype(np.uint32)
        got = selected(mem, q, ids, None, 2, kind, 0.1)
        mem.lay, mem.cache, mem.tables = small
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_selected_rows_of_hidden_pages_and_nan(torch):
    rng = np.random.default_rng(21)

    def spoil(mem, k, v):
        v[20, 0, 40] = np.nan
        k[150, 1, 3] = np.nan
    mem = Memory(torch, rng, [100, 90], 64, 2, 16, spoil=spoil)
    mem.tables[0, 4] = mem.pages
    ids = np.stack([np.stack([rng.permutation(90)[:40] for _ in range(2)]) for _ in range(2)]).astype(np.uint64)
    ids[0, 0, 3], ids[1, 0, 5] = 20, 20
    ids[0, 1, 0], ids[1, 1, 0] = 50, 50
    q, qx = as_type(torch, rng.standard_normal((2, 4, 64)), "bf16")
    got, lse = selected(mem, q, ids, None, 2, "bf16", 0.3)
    check_selected(mem, got, lse, qx, ids, None, 2, "bf16", float(np.float32(0.3)), there=lambda i, t: not (i == 0 and t // 16 == 4))


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_selected_values_near_the_largest_stay_finite(torch, kind, d):
    lengths = [300, 90]
    mem, q, qx, _ = check_sizes(torch, lengths, [1, 1], d, 2, 2, kind, True)
    ids = np.stack([np.stack([np.arange(300) % t for t in lengths]) for _ in range(2)]).astype(np.uint64)
    scale = 1.0 / np.sqrt(d)
    got, lse = selected(mem, q, ids, None, 2, kind, scale)
    check_selected(mem, got, lse, qx, ids, None, 2, kind, float(np.float32(scale)))


def test_lists_of_no_rows(torch):
    rng = np.random.default_rng(23)
    mem = Memory(torch, rng, [40, 0], 64, 2, 16)
    q, _ = as_type(torch, rng.standard_normal((2, 4, 64)), "bf16")
    for ids, counts in ((np.zeros((2, 2, 0), np.uint64), None), (np.full((2, 2, 5), 2**64 - 1, np.uint64), None), (np.zeros((2, 2, 5), np.uint64), np.zeros((2, 2)))):
        got, lse = selected(mem, q, ids, counts, 2, "bf16", 0.3)
        assert (got[:2] == 0).all() and np.isneginf(lse[:2]).all()


def test_selecting_every_row_is_attending_to_all(torch):
    rng = np.random.default_rng(22)
    mem = Memory(torch, rng, [130, 64], 128, 2, 16)
    q, qx = as_type(torch, rng.standard_normal((2, 8, 128)), "fp32")
    ids = np.tile(np.arange(130, dtype=np.uint64), (2, 2, 1))
    got, lse = selected(mem, q, ids, None, 4, "fp32", 0.1)
    want, wl, _ = attend(mem, q, [1, 1], 4, "fp32", False, 0.1)
    for i in range(2):
        for h in range(8):
            _, _, bo, bl = ref.attend_row(qx[i, h], mem.k[mem.rows_of(i)][:, h // 4], mem.v[mem.rows_of(i)][:, h // 4], float(np.float32(0.1)), "fp32")
            assert (np.abs(got[i, h] - want[i, h]) <= 2 * bo).all() and abs(lse[i, h] - wl[i, h]) <= 2 * bl


# ---- calls of more threads than a launch takes in one direction -------------------------------------------------------------------

def test_more_rows_than_a_launch_has_threads_in_a_row(torch):
    """Append and read of 2^29 + 77 tokens, eight threads to a row; a few of them have slots, at both ends."""
    import zvdb_amd as zv
    n, d = 2**29 + 77, 8
    lay = zv.KVLayout(head_dim=d, kv_heads=1, page_size=16, pages=16)
    slots = torch.full((n,), -1, dtype=torch.int64, device="cuda")
    slots[:100], slots[-100:] = torch.arange(100, device="cuda"), torch.arange(100, 200, device="cuda")
    k = torch.zeros((n, d), dtype=torch.bfloat16, device="cuda")
    k[:100], k[-100:] = (torch.randn(100, d, device="cuda") for _ in range(2))
    few, rows = torch.cat((slots[:100], slots[-100:])), torch.cat((k[:100], k[-100:]))
    cache, want = (torch.zeros(lay.pages * lay.page_bytes, dtype=torch.uint8, device="cuda") for _ in range(2))
    lay.append_dev(cache.data_ptr(), k.data_ptr(), d, k.data_ptr(), d, zv.KV_BF16, n, slots.data_ptr(), stream(torch))
    lay.append_dev(want.data_ptr(), rows.data_ptr(), d, rows.data_ptr(), d, zv.KV_BF16, 200, few.data_ptr(), stream(torch))
    assert torch.equal(cache, want)
    a, b = torch.empty_like(rows), torch.empty_like(rows)
    lay.read_dev(want.data_ptr(), few.data_ptr(), 200, a.data_ptr(), b.data_ptr(), zv.KV_BF16, stream(torch))
    out = k.fill_(3.0)
    for at in ((out.data_ptr(), 0), (0, out.data_ptr())):
        out.fill_(3.0)
        lay.read_dev(cache.data_ptr(), slots.data_ptr(), n, *at, zv.KV_BF16, stream(torch))
        assert torch.equal(torch.cat((out[:100], out[-100:])), a if at[0] else b) and not out[100:-100].any()


@pytest.mark.parametrize("n,heads,group,max_new", [(2**21 + 3, 8, 1, 1), (16_384, 8, 8, 2_064)])  # single tokens; one long prompt among them
def test_more_requests_than_a_launch_has_threads_in_a_row(torch, n, heads, group, max_new):
    """One memory that all requests read, each some of its tokens; halves of the call are bit for bit the same."""
    import zvdb_amd as zv
    d, qh, typ = 64, heads * group, kv_type("bf16")
    rng = np.random.default_rng(51)
    mem = Memory(torch, rng, [max_new + 40], d, heads, 16)
    gen = torch.Generator("cuda").manual_seed(52)
    new = torch.ones(n, dtype=torch.int32, device="cuda")
    new[n // 3] = max_new
    lengths = new + torch.randint(0, 40, (n,), generator=gen, device="cuda", dtype=torch.int32)
    starts = torch.cat((new.new_zeros(1), torch.cumsum(new, 0).int()))
    tables = mem.i32(mem.tables).expand(n, -1).contiguous()
    rows, max_length = int(starts[-1]), max_new + 40
    q = torch.randn((rows, qh, d), generator=gen, device="cuda").to(torch.bfloat16)

    def call(first, last):
        at, to = int(starts[first]), int(starts[last])
        out = torch.full((to - at + 1, qh, d), 77.0, dtype=torch.bfloat16, device="cuda")
        lse = torch.full((to - at + 1, qh), 77.0, device="cuda")
        own = starts[first:last + 1] - starts[first]
        assert mem.lay.attend_workspace(typ, qh, last - first, to - at, max_new, max_length) == 0
        mem.lay.attend_dev(mem.cache.data_ptr(), q[at:].data_ptr(), qh * d, typ, qh, last - first, own.data_ptr(), to - at, max_new, lengths[first:].data_ptr(),
                           tables[first:].data_ptr(), mem.stride, max_length, 0.125, True, 0, 0, out.data_ptr(), lse.data_ptr(), stream(torch))
        torch.cuda.synchronize()
        assert (out[-1] == 77.0).all() and (lse[-1] == 77.0).all()
        return out[:-1], lse[:-1]

    whole, parts = call(0, n), [call(0, n // 2), call(n // 2, n)]
    for x, y in zip(whole, zip(*parts)):
        assert torch.equal(x, torch.cat(y))
    for i in (0, n // 3, n - 1):  # and some rows against the definition
        r, length = int(starts[i + 1]) - 1, int(lengths[i])
        for h in (0, qh - 1):
            o, l, bo, bl = ref.attend_row(q[r, h].double().cpu().numpy(), mem.k[:length, h // group], mem.v[:length, h // group], 0.125, "bf16")
            assert (np.abs(whole[0][r, h].double().cpu().numpy() - o) <= bo).all() and abs(float(whole[1][r, h]) - l) <= bl


def test_more_lists_than_a_launch_has_threads_in_a_row(torch):
    n, heads, d, k = 2**21 + 3, 8, 64, 2
    mem = Memory(torch, np.random.default_rng(53), [60], d, heads, 16)
    gen = torch.Generator("cuda").manual_seed(54)
    q = torch.randn((n, heads, d), generator=gen, device="cuda").to(torch.bfloat16)
    ids = torch.randint(0, 60, (heads, n, k), generator=gen, device="cuda")
    lengths, tables = torch.full((n,), 60, dtype=torch.int32, device="cuda"), mem.i32(mem.tables).expand(n, -1).contiguous()

    def call(first, last):
        m, own = last - first, ids[:, first:last].contiguous()
        out = torch.full((m + 1, heads, d), 77.0, dtype=torch.bfloat16, device="cuda")
        lse = torch.full((m + 1, heads), 77.0, device="cuda")
        mem.lay.attend_selected_dev(mem.cache.data_ptr(), q[first:].data_ptr(), heads * d, kv_type("bf16"), heads, m, own.data_ptr(), 0, k, lengths.data_ptr(), tables.data_ptr(),
                                    mem.stride, 0.125, out.data_ptr(), lse.data_ptr(), stream(torch))
        torch.cuda.synchronize()
        assert (out[-1] == 77.0).all() and (lse[-1] == 77.0).all()
        return out[:-1], lse[:-1]

    whole, parts = call(0, n), [call(0, n // 2), call(n // 2, n)]
    for x, y in zip(whole, zip(*parts)):
        assert torch.equal(x, torch.cat(y)) and torch.isfinite(x).all()


# ---- the calls together -----------------------------------------------------------------------------------------------------------

class Server:
    """A decode loop as a program runs it: plan, append, attend on a stream; lengths, cursor and tables stay on the device."""

    def __init__(self, torch, n, d, heads, group, page, slot_cap, max_length, kind="bf16"):
        import zvdb_amd as zv
        self.torch, self.n, self.d, self.heads, self.group, self.kind, self.cap, self.max_length = torch, n, d, heads, group, kind, slot_cap, max_length
        self.stride = -(-max_length // page)
        pages = n * self.stride
        self.lay = zv.KVLayout(head_dim=d, kv_heads=heads, page_size=page, pages=pages)
        dev = dict(device="cuda")
        i32 = dict(dtype=torch.int32, **dev)
        self.cache = torch.full((pages * self.lay.page_bytes,), 255, dtype=torch.uint8, **dev)
        self.ring = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
        self.cursor, self.next_cursor = torch.tensor([0, pages], dtype=torch.int64, **dev), torch.zeros(2, dtype=torch.int64, **dev)
        self.lengths, self.next_lengths, self.new = torch.zeros(n, **i32), torch.zeros(n, **i32), torch.zeros(n, **i32)
        self.tables = torch.full((n, self.stride), -1, **i32)
        self.starts, self.status = torch.zeros(n + 1, **i32), torch.zeros(4, **i32)
        self.slots = torch.zeros(slot_cap, dtype=torch.int64, **dev)
        dt = torch.bfloat16 if kind == "bf16" else torch.float32
        self.qkv = torch.zeros(slot_cap, (heads * group + 2 * heads) * d, dtype=dt, **dev)  # one projection's rows: q, k, v side by side
        self.out = torch.zeros(slot_cap, heads * group, d, dtype=dt, **dev)
        self.lse = torch.zeros(slot_cap, heads * group, **dev)
        self.ws = torch.empty(max(16, self.lay.attend_workspace(kv_type(kind), heads * group, n, slot_cap, slot_cap, max_length)), dtype=torch.uint8, **dev)

    def step(self):
        s, lay, row, size = stream(self.torch), self.lay, self.qkv.shape[1], self.qkv.element_size()
        q, k = self.qkv.data_ptr(), self.qkv.data_ptr() + self.heads * self.group * self.d * size
        v = k + self.heads * self.d * size
        lay.plan_dev(self.lengths.data_ptr(), self.new.data_ptr(), self.n, self.ring.data_ptr(), self.ring.numel(), self.cursor.data_ptr(), self.tables.data_ptr(),
                     self.stride, self.starts.data_ptr(), self.slots.data_ptr(), self.cap, self.next_lengths.data_ptr(), self.next_cursor.data_ptr(),
                     self.status.data_ptr(), s)
        lay.append_dev(self.cache.data_ptr(), k, row, v, row, kv_type(self.kind), self.cap, self.slots.data_ptr(), s)
        lay.attend_dev(self.cache.data_ptr(), q, row, kv_type(self.kind), self.heads * self.group, self.n, self.starts.data_ptr(), self.cap, self.cap,
                       self.next_lengths.data_ptr(), self.tables.data_ptr(), self.stride, self.max_length, 0.17, True, self.ws.data_ptr(), self.ws.numel(),
                       self.out.data_ptr(), self.lse.data_ptr(), s)
        self.lengths.copy_(self.next_lengths)
        self.cursor.copy_(self.next_cursor)


def serve_and_check(torch, server, rounds, run, rng):
    """rounds: new tokens of each request, step by step; every row of every step against the restatement."""
    n, d, heads, group = server.n, server.d, server.heads, server.group
    keys, vals = [np.zeros((0, heads, d)) for _ in range(n)], [np.zeros((0, heads, d)) for _ in range(n)]
    scale = float(np.float32(0.17))
    for new in rounds:
        total = sum(new)
        x, xx = as_type(torch, rng.standard_normal((server.cap, server.qkv.shape[1])) * 1.3, server.kind)
        server.qkv.copy_(x)
        server.new.copy_(torch.tensor(new, dtype=torch.int32))
        run()
        torch.cuda.synchronize()
        assert server.status.tolist()[0] == 0 and server.starts.tolist()[-1] == total
        got, lse = server.out.double().cpu().numpy(), server.lse.double().cpu().numpy()
        at = 0
        for i, m in enumerate(new):
            part = xx[at:at + m]
            qw, kw = heads * group * d, heads * d
            for store, rows in ((keys, part[:, qw:qw + kw]), (vals, part[:, qw + kw:])):
                rows = rows.reshape(m, heads, d)
                store[i] = np.concatenate([store[i], np.stack([ref.encode_rows(rows[:, h], d)[2] for h in range(heads)], 1)]) if m else store[i]
            for j in range(m):
                see = len(keys[i]) - m + j + 1
                for h in range(heads * group):
                    o, l, bo, bl = ref.attend_row(part[j, h * d:(h + 1) * d], keys[i][:see, h // group], vals[i][:see, h // group], scale, server.kind)
                    assert (np.abs(got[at + j, h] - o) <= bo).all() and abs(lse[at + j, h] - l) <= bl, (i, j, h)
            at += m
    return [len(k) for k in keys]


ROUNDS = [[5, 0, 17, 1], [1, 1, 1, 1], [1, 0, 1, 1], [3, 2, 0, 30], [1, 1, 1, 1], [0, 0, 0, 0], [16, 1, 1, 7], [1, 1, 1, 1]]


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("d,heads,group,page", [(64, 2, 2, 16), (128, 1, 3, 32)])
def test_serving_step_by_step(torch, kind, d, heads, group, page):
    server = Server(torch, 4, d, heads, group, page, 36, 128, kind)
    lengths = serve_and_check(torch, server, ROUNDS, server.step, np.random.default_rng(31))
    assert server.lengths.tolist() == lengths


def test_serving_on_another_stream(torch):
    server = Server(torch, 4, 64, 2, 2, 16, 36, 128)
    other = torch.cuda.Stream()

    def run():
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            server.step()
        torch.cuda.current_stream().wait_stream(other)
    serve_and_check(torch, server, ROUNDS, run, np.random.default_rng(32))


@pytest.mark.parametrize("max_length", [128, 4096])  # the second is split: workspace and join in the graph
def test_serving_from_a_graph(torch, max_length):
    """The step captured once and replayed for every round, whatever the lengths are; other work of the program in between."""
    server = Server(torch, 4, 64, 2, 2, 16, 36, max_length)
    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm):
        server.step()  # no new tokens: nothing changes
    warm.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        server.step()
    noise = torch.randn(512, 512, device="cuda")

    def run():
        graph.replay()
        torch.cuda.synchronize()
        (noise @ noise).sum().item()
    serve_and_check(torch, server, ROUNDS, run, np.random.default_rng(33))


def test_two_servers_on_two_streams(torch):
    """Two caches with workspaces of their own, their steps in flight together."""
    servers, streams = [Server(torch, 4, 64, 1, 4, 16, 36, 2048) for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    alone = [Server(torch, 4, 64, 1, 4, 16, 36, 2048) for _ in range(2)]
    rng = np.random.default_rng(34)
    for new in ROUNDS:
        for x, y in zip(servers, alone):
            x.qkv.copy_(as_type(torch, rng.standard_normal(tuple(x.qkv.shape)), "bf16")[0])
            y.qkv.copy_(x.qkv)
            for z in (x, y):
                z.new.copy_(torch.tensor(new, dtype=torch.int32))
        torch.cuda.synchronize()
        for x, s in zip(servers, streams):
            with torch.cuda.stream(s):
                x.step()
        torch.cuda.synchronize()
        for x, y in zip(servers, alone):
            y.step()
            torch.cuda.synchronize()
            total = sum(new)
            assert torch.equal(x.out[:total], y.out[:total]) and torch.equal(x.lse[:total], y.lse[:total]) and torch.equal(x.cache, y.cache)


def test_a_full_ring_stops_the_step_and_nothing_else(torch):
    server = Server(torch, 2, 64, 1, 1, 16, 40, 64)
    server.new.copy_(torch.tensor([20, 20], dtype=torch.int32))
    server.step()                            # two pages each
    server.cursor[1] = server.cursor[0] + 1  # one left
    server.new.copy_(torch.tensor([20, 20], dtype=torch.int32))  # 40 tokens: a page more for each
    before = [t.clone() for t in (server.cache, server.tables, server.lengths, server.cursor)]
    server.out.fill_(9.0)
    server.step()
    torch.cuda.synchronize()
    assert server.status.tolist() == [1, 2, 40, 0]
    assert all(torch.equal(a, b) for a, b in zip(before, (server.cache, server.tables, server.lengths, server.cursor))) and (server.out == 9.0).all()
    server.new.copy_(torch.tensor([20, 0], dtype=torch.int32))   # the one that is left is enough for one of them
    server.step()
    torch.cuda.synchronize()
    assert server.status.tolist() == [0, 1, 20, 0] and server.lengths.tolist() == [40, 20] and (server.out[:20] != 9.0).any() and (server.out[20:] == 9.0).all()


@pytest.mark.parametrize("mode", ["f32", "bf16"])
def test_searching_an_index_and_attending_to_what_it_found(torch, mode):
    """Keys of each head in an index of the framework (dot product), its search's ids and counts straight into the attention over the
    same tokens' keys and values in 4 bits."""
    import zvdb_amd as zv
    rng = np.random.default_rng(41)
    tokens, d, heads, n, k = 900, 64, 2, 5, 12
    mem = Memory(torch, rng, [tokens], d, heads, 16)
    mem.lengths, mem.tables = [tokens] * n, np.repeat(mem.tables, n, 0)   # one memory that every request reads
    q, qx = as_type(torch, rng.standard_normal((n, heads, d)), "fp32")
    ids = torch.zeros((heads, n, k), dtype=torch.int64, device="cuda")
    dist = torch.zeros((heads, n, k), dtype=torch.float32, device="cuda")
    counts = torch.zeros((heads, n), dtype=torch.int32, device="cuda")
    m, s, keep = zv.BF_F32 if mode == "f32" else zv.BF_BF16, stream(torch), []
    for h in range(heads):
        idx = zv.Index(dim=d, metric=zv.METRIC_DOT, capacity=tokens, flags=zv.FLAG_BF16_MIRROR)
        idx.add(mem.k[:, h].astype(np.float32))
        wsb = idx.bruteforce_workspace(n, k, m)
        ws, qh = torch.empty(wsb, dtype=torch.uint8, device="cuda"), q[:, h].contiguous()
        idx.search_bruteforce_dev(qh.data_ptr(), n, d, k, m, 0, ws.data_ptr(), wsb, ids[h].data_ptr(), dist[h].data_ptr(), counts[h].data_ptr(), s)
        keep += [idx, ws, qh]
    out, lse = torch.zeros_like(q), torch.zeros((n, heads), device="cuda")
    L, T = mem.i32(mem.lengths), mem.i32(mem.tables)
    mem.lay.attend_selected_dev(mem.cache.data_ptr(), q.data_ptr(), heads * d, zv.KV_F32, heads, n, ids.data_ptr(), counts.data_ptr(), k, L.data_ptr(), T.data_ptr(),
                                mem.stride, 0.125, out.data_ptr(), lse.data_ptr(), s)
    torch.cuda.synchronize()
    got, gl = out.double().cpu().numpy(), lse.double().cpu().numpy()
    for i in range(n):
        for h in range(heads):
            best = np.argsort(-(mem.k[:, h] @ qx[i, h]), kind="stable")[:k]
            assert set(best.tolist()) == set(ids[h, i].tolist()) and counts[h, i] == k
            o, l, bo, bl = ref.attend_row(qx[i, h], mem.k[best, h], mem.v[best, h], 0.125, "fp32")
            assert (np.abs(got[i, h] - o) <= bo).all() and abs(gl[i, h] - l) <= bl


@pytest.mark.parametrize("max_new,max_length,split", [(300, 700, False), (100, 1500, True)])
def test_prompts_from_a_graph(torch, max_new, max_length, split):
    """Prompts captured once; lengths and row starts change on the device between the replays, and with them which blocks have tiles."""
    heads, group, d, n, page = (16, 2, 64, 6, 16) if not split else (2, 3, 64, 6, 16)
    qh, rows = heads * group, 2 * max_new
    mem = Memory(torch, np.random.default_rng(41), [max_length] * n, d, heads, page)
    q, _ = as_type(torch, np.random.default_rng(42).standard_normal((rows, qh, d)), "bf16")
    typ = kv_type("bf16")
    size = mem.lay.attend_workspace(typ, qh, n, rows, max_new, max_length)
    assert (size > 0) == split
    ws = torch.full((max(size, 16),), 255, dtype=torch.uint8, device="cuda")
    tables, starts, lengths = mem.i32(mem.tables), mem.i32([0] * (n + 1)), mem.i32([0] * n)
    out, lse = torch.empty((rows, qh, d), dtype=torch.bfloat16, device="cuda"), torch.empty((rows, qh), device="cuda")

    def call():
        mem.lay.attend_dev(mem.cache.data_ptr(), q.data_ptr(), qh * d, typ, qh, n, starts.data_ptr(), rows, max_new, lengths.data_ptr(), tables.data_ptr(),
                           mem.stride, max_length, 0.125, True, ws.data_ptr(), size, out.data_ptr(), lse.data_ptr(), stream(torch))

    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm):
        call()
    warm.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    rng = np.random.default_rng(43)
    for new in ([max_new, 0, 17, 1, 90, 30], [0] * n, [1] * n, [5, max_new, 60, 0, 0, max_new // 2], [64, 64, 0, 65, 63, 1]):
        starts.copy_(mem.i32(np.concatenate(([0], np.cumsum(new)))))
        lengths.copy_(mem.i32([x + int(rng.integers(0, max_length - x + 1)) for x in new]))
        out.fill_(77.0), lse.fill_(77.0)
        call()
        torch.cuda.synchronize()
        want = out.clone(), lse.clone()
        assert (want[0][:sum(new)] != 77.0).all() and (want[0][sum(new):] == 77.0).all() and torch.isfinite(want[1][:sum(new)]).all()
        for _ in range(3):
            out.fill_(77.0), lse.fill_(77.0), ws.fill_(255)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
