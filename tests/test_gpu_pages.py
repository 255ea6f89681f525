"""The paged 4-bit cache (s2hip.PagedKv) against 64-bit computations and plain Python:
sizes around the pages' and tiles' borders, shared pages, values that must not be
seen, rows of pages made anew, pools compacted, graphs and streams."""

import math
import random

import numpy as np
import pytest
import torch

import kv_util
import pages_util
from s2hip import KvOps, PagedKv, S2HipError, rope_frequencies
from s2hip.pages import ERR_FULL, ERR_LENS, ERR_PAGE, ERR_POSITION, ERR_RANGE, ERR_REFS

pytestmark = pytest.mark.gpu
U = kv_util.U


@pytest.fixture(autouse=True)
def float32_tensors():
    """Whatever another module has made the default type."""
    was = torch.get_default_dtype()
    torch.set_default_dtype(torch.float32)
    yield
    torch.set_default_dtype(was)


SHAPES = {"gqa4": (32, 8, 128), "tiny": (8, 2, 64), "mha": (4, 4, 64), "gqa3": (6, 2, 128), "gqa7": (14, 2, 128), "wide": (64, 1, 64)}


def dev(x, dtype=torch.int32):
    return torch.as_tensor(x, dtype=dtype).cuda()


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, spread=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * spread


def stream():
    return torch.cuda.current_stream().cuda_stream


def ptr(x):
    return 0 if x is None else x.data_ptr()


def rows_of(lens, page, width, order, shared=0):
    """A table whose rows take pages from `order`; the first `shared` pages of all rows are the same."""
    table, at = [], shared
    for n in lens:
        row = []
        for i in range(-(-n // page)):
            if i < shared:
                row.append(order[i])
            else:
                row.append(order[at])
                at += 1
        table.append(row + [-1] * (width - len(row)))
    return table, at


class Pool:
    """Random pages, the rows of a batch, and the call's arrays."""

    def __init__(self, shape, page, lens, new, shared=0, rows=None, seed=0, spread=1.5, width=None, spare=3, **kw):
        self.H, self.G, self.hd = shape
        self.page, self.R, self.n = page, len(lens), rows or max(1, max(new))
        self.lens_h, self.new_h = list(lens), list(new)
        self.width = width or max(1, max(-(-n // page) for n in lens)) + 1
        self.lay = pages_util.Layout(page, self.hd)
        count = shared + sum(max(0, -(-n // page) - shared) for n in lens) + spare
        order = list(range(count))
        random.Random(seed).shuffle(order)
        self.pages = count
        self.table_h, self.taken = rows_of(lens, page, self.width, order, shared)
        self.order = order
        r = np.random.default_rng(seed)
        part = r.integers(0, 256, (count, self.G, self.lay.part), dtype=np.uint8)
        d = (r.standard_normal((count, self.G, 2 * page * self.hd // 32)) * 0.15).astype(np.float16)
        d = np.array([pages_util.d8(float(x)) for x in d.ravel()], np.float16).reshape(d.shape)
        part[:, :, page * self.hd :] = d.view(np.uint8).reshape(count, self.G, -1)
        self.pool_h = part
        self.pool = torch.from_numpy(part).cuda()
        self.table, self.lens, self.new = dev(self.table_h), dev(lens), dev(new)
        g = gen(seed)
        self.q = normal(g, self.R, self.n, self.H, self.hd, spread=spread)
        self.out = torch.full_like(self.q, 7.0)
        self.ops = PagedKv(self.H, self.G, self.hd, page, count, self.width, max_requests=max(self.R, 1), max_tokens=self.R * self.n, **kw)
        assert self.ops.page_bytes == self.G * self.lay.part

    def view(self):
        return self.ops.view(ptr(self.pool), ptr(self.table), ptr(self.lens), self.R, new_lens=ptr(self.new))

    def dense(self):
        """Keys and values [R][G][cap][hd] that the rows hold, zeros elsewhere."""
        cap = max(1, max(-(-n // self.page) for n in self.lens_h)) * self.page
        k = np.zeros((self.R, self.G, cap, self.hd))
        v = np.zeros_like(k)
        pool = self.pool.cpu().numpy()
        for b in range(self.R):
            for i in range(-(-self.lens_h[b] // self.page)):
                p = self.table_h[b][i]
                if 0 <= p < self.pages:
                    kk, vv = self.lay.read(pool[p])
                    k[b, :, i * self.page : (i + 1) * self.page], v[b, :, i * self.page : (i + 1) * self.page] = kk, vv
        return torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()

    def attend(self):
        self.ops.attend(self.view(), ptr(self.q), self.n, ptr(self.out), stream=stream())
        torch.cuda.synchronize()
        return self.out

    def expect(self):
        k, v = self.dense()
        return kv_util.attend(self.q, k, v, self.lens_h, self.new_h)

    def check(self, out, want=None):
        ref, tol = (want or self.expect())[:2]
        live = torch.arange(self.n, device="cuda")[None] < self.new[:, None]
        assert bool((out[~live] == 7.0).all()), "rows of no token were written"
        if not bool(live.any()):
            return
        far = (out.double() - ref).abs()[live]
        assert bool((far <= tol[live]).all()), f"off by {far.max().item():.3g}, {(far / tol[live]).max().item():.3g} of the bound"

    def check_all(self):
        self.check(self.attend())
        assert self.ops.errors(stream()) == 0


# --------------------------------------------------------------------------
# attend
# --------------------------------------------------------------------------
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_attend_step(shape, page):
    Pool(SHAPES[shape], page, [1, 2, 15, 16, 17, 33, 100], [1] * 7, seed=page).check_all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 3001])
def test_attend_lengths(length, hd):
    Pool((8, 2, hd), (16, 32, 64, 128)[length % 4], [length], [1], seed=length).check_all()


@pytest.mark.parametrize("requests", [1, 2, 4, 5, 8, 9, 16, 17])
def test_attend_shared_pages(requests):
    """Rows that begin alike and go on apart."""
    lens = [333 + 1 + (37 * b) % 90 for b in range(requests)]
    Pool((32, 8, 128), 32, lens, [1] * requests, shared=10, seed=requests).check_all()


@pytest.mark.parametrize("page", [16, 64])
def test_attend_rows_all_the_same(page):
    p = Pool((8, 2, 128), page, [200] * 6, [1] * 6, shared=-(-200 // page), seed=3)
    p.check_all()


# Rows of the table as long as the lengths need, and so long that a call counts as much work (it is launched by them)
ROOM = [None, 32768, 131072]


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("n", [2, 3, 4, 5, 7, 8, 9, 16, 31, 32, 33, 64, 65, 130])
def test_attend_several_tokens(n, page, room):
    """Causal within the new tokens; ragged; an idle request between others."""
    new = [n, max(1, n // 2), 0, 1, n]
    lens = [n, n // 2 + 40, 9, 1, n + 77]
    Pool((8, 2, 128), page, lens, new, seed=n, width=room and room // page).check_all()


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("shape,requests,n,length,shared", [
    ((32, 8, 128), 2, 200, 63, 0), ((32, 8, 128), 1, 500, 0, 0), ((32, 8, 128), 2, 130, 1000, 15), ((8, 2, 64), 3, 300, 700, 10), ((16, 16, 64), 2, 257, 100, 0),
    ((14, 2, 128), 2, 150, 300, 4), ((32, 8, 128), 5, 40, 800, 12), ((64, 1, 64), 2, 40, 300, 2), ((6, 2, 128), 9, 33, 129, 2)])
def test_attend_turns(shape, requests, n, length, shared, room):
    new = [max(1, n - 13 * b) for b in range(requests)]
    Pool(shape, 64, [length + x for x in new], new, shared=shared, seed=n, width=room and room // 64).check_all()


@pytest.mark.parametrize("room", ROOM[1:])
@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("extra", [0, 1, 14, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 127, 128, 129])
def test_attend_turn_borders(extra, hd, page, room):
    """Turns that begin and end around the borders of tiles and pages."""
    Pool((8, 2, hd), page, [32 + extra, 64 + extra, 33], [32, 9, 33], seed=extra, width=room // page).check_all()


@pytest.mark.parametrize("shared", [0, 5])
@pytest.mark.parametrize("n", [31, 32, 33, 63, 64, 65, 95, 96, 97])
def test_attend_row_tiles(n, shared):
    """Row tiles of one request each, or of several, by how many rows a request has; idle ones among them."""
    new = [n, 1, 0, n, n - 1, n // 2, n]
    Pool((8, 2, 64), 32, [shared * 32 + x + 10 * i if x else 0 for i, x in enumerate(new)], new, shared=shared, seed=n, width=4096).check_all()
    new = [n // 2, n // 2, 0, 1, n // 4, n // 2, n // 2, n // 2, n // 2]
    Pool((4, 2, 128), 64, [shared * 64 + x + 10 * i if x else 0 for i, x in enumerate(new)], new, shared=shared, seed=n, width=4096).check_all()


@pytest.mark.parametrize("shared", [0, 3])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [3, 4, 5, 6, 7, 8, 9, 11, 12, 13, 17, 23])
def test_attend_speculative_steps(n, hd, page, shared):
    """A few tokens of each request, in tables with room for long runs: row tiles of 16 and 32."""
    new = [n, 1, 0, n, n - 1, n // 2, n]
    lens = [shared * page + x + 70 * i if x else 0 for i, x in enumerate(new)]
    Pool((8, 2, hd), page, lens, new, shared=shared, seed=n, width=131072 // page).check_all()
    new, lens = new[:2], [lens[0] + 3000, lens[1]]
    Pool((8, 2, hd), page, lens, new, shared=shared, seed=n, rows=n, width=16384 // page).check_all()


def test_attend_many_requests():
    g = random.Random(1)
    lens = [g.randint(0, 120) for _ in range(200)]
    Pool((8, 2, 64), 16, lens, [min(1, n) for n in lens], seed=1).check_all()


@pytest.mark.parametrize("shape", ["gqa4", "tiny"])
def test_attend_long(shape):
    Pool(SHAPES[shape], 128, [20001, 3, 9000], [1, 1, 1], seed=2).check_all()


def test_attend_drawn():
    """Sizes, pages and lengths at random, many of them."""
    g = random.Random(77)
    for i in range(60):
        shape = g.choice(list(SHAPES.values()))
        requests = g.randint(1, 9)
        n = g.choice([1, 1, 1, 2, 3, 5, 17, 60, 100])
        new = [g.randint(0, n) for _ in range(requests)]
        shared = g.choice([0, 0, g.randint(1, 6)])
        page = g.choice([16, 32, 64, 128])
        lens = [shared * page + x + g.choice([0, 1, g.randint(0, 40), g.randint(0, 400)]) if x else 0 for x in new]
        width = g.choice([None, 40000 // page])
        print(i, shape, page, shared, lens, new, width, flush=True)
        Pool(shape, page, lens, new, shared=shared, rows=n, seed=i, width=width).check_all()


def test_attend_without_new_lens():
    p = Pool((8, 2, 128), 32, [5, 0, 40], [2, 0, 2], seed=4)
    p.ops.attend(p.ops.view(ptr(p.pool), ptr(p.table), ptr(p.lens), 3), ptr(p.q), 2, ptr(p.out), stream=stream())
    torch.cuda.synchronize()
    p.check(p.out)
    assert p.ops.errors(stream()) == 0


@pytest.mark.parametrize("room", [None, 1000, 4000])
@pytest.mark.parametrize("n", [1, 3, 40])
@pytest.mark.parametrize("hd", [64, 128])
def test_attend_never_sees_the_rest(n, hd, room):
    """Slots behind the last token, pages of no row and table entries behind a row may hold anything: no bit changes."""
    lens = [n + 21, n, n + 90]
    p = Pool((8, 2, hd), 32, lens, [n, n, max(1, n - 1)], seed=n, width=room or 7)
    want = p.attend().clone()
    p.check(want)
    for fill in (0xFF, 0x7C, 0x00):
        pool = np.full_like(p.pool_h, fill)
        for b, length in enumerate(lens):
            for s in range(length):
                at, s0 = p.table_h[b][s // 32], s % 32
                for (bits, _), scale in ((p.lay.key, p.lay.key_scale), (p.lay.value, p.lay.value_scale)):
                    for places in (bits[s0], scale[s0], scale[s0] + 1):
                        pool[at][:, places] = p.pool_h[at][:, places]
        p.pool.copy_(torch.from_numpy(pool))
        table = [[x if x >= 0 else (1 << 30 if fill else -5) for x in row] for row in p.table_h]
        p.table.copy_(dev(table))
        p.out.fill_(7.0)
        assert torch.equal(p.attend(), want)
    assert p.ops.errors(stream()) == 0


@pytest.mark.parametrize("part", ["key", "value"])
@pytest.mark.parametrize("room", [None, 2000])
@pytest.mark.parametrize("n", [1, 5, 40])
def test_attend_no_number_reaches_who_sees_it(part, n, room):
    """A block of no numbers in one slot: rows that see it, and no others."""
    length = n + 30
    p = Pool((8, 2, 128), 16, [length, length], [n, n], seed=n, width=room)
    slot, g, group = length - max(1, n // 2), 1, 2  # of request 1
    clean = p.attend().clone()
    p.check(clean)
    at = (p.lay.key_scale if part == "key" else p.lay.value_scale)[slot % 16, group]
    pool = p.pool_h.copy()
    pool[p.table_h[1][slot // 16], g, at : at + 2] = np.array([math.nan], np.float16).view(np.uint8)
    p.pool.copy_(torch.from_numpy(pool))
    p.out.fill_(7.0)
    out = p.attend()
    hit = torch.zeros(2, n, 8, 128, dtype=torch.bool, device="cuda")
    t0 = slot - (length - n)
    dims = slice(None) if part == "key" else slice(32 * group, 32 * group + 32)
    hit[1, max(0, t0) :, 4 * g : 4 * g + 4, dims] = True
    assert bool(out[hit].isnan().all())
    assert bool((out[~hit] == clean[~hit]).all()) if part == "value" else bool(torch.isfinite(out[~hit]).all())
    p.check(torch.where(hit, clean, out), kv_util.attend(p.q, *_without(p, pool), p.lens_h, p.new_h))


def _without(p, pool):
    clean = p.pool
    p.pool = torch.from_numpy(p.pool_h).cuda()
    k, v = p.dense()
    p.pool = clean
    return k, v


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("part", ["key", "value"])
@pytest.mark.parametrize("room", [None, 4000])
@pytest.mark.parametrize("n", [1, 5, 40])
def test_attend_scales_beyond_the_format(n, room, part, hd):
    """A finite scale that append never writes, in a slot of one request: rows that do not see it (its earlier tokens, and other
    requests, before and behind it in a row tile) keep every bit."""
    length, g, group = n + 40, 1, 1
    p = Pool((8, 2, hd), 16, [length] * 3, [n] * 3, seed=n, width=room)
    clean = p.attend().clone()
    p.check(clean)
    dims = slice(None) if part == "key" else slice(32 * group, 32 * group + 32)
    for slot in (3, length - max(1, n // 2)):  # of request 1: in a tile that its rows see whole, and among the new ones
        at = (p.lay.key_scale if part == "key" else p.lay.value_scale)[slot % 16, group]
        hit = torch.zeros(3, n, 8, hd, dtype=torch.bool, device="cuda")
        hit[1, max(0, slot - (length - n)) :, 4 * g : 4 * g + 4, dims] = True
        for bits in (0x6801, 0x6955, 0x6C00, 0x7800, 0x7BFF, 0xF800, 0xE801):
            pool = p.pool_h.copy()
            pool[p.table_h[1][slot // 16], g, at : at + 2] = np.array([bits], np.uint16).view(np.uint8)
            p.pool.copy_(torch.from_numpy(pool))
            p.out.fill_(7.0)
            out = p.attend()
            assert torch.equal(out[~hit], clean[~hit]), (slot, hex(bits))
    assert p.ops.errors(stream()) == 0


@pytest.mark.parametrize("n", [3, 40])
def test_attend_query_of_no_number(n):
    p = Pool((8, 2, 128), 16, [50, 50], [n, n], seed=9, width=2000)
    clean = p.attend().clone()
    p.q[1, 1, 5, 17] = math.nan
    p.q[0, 2, 0, 3] = math.inf
    p.out.fill_(7.0)
    out = p.attend()
    assert bool(out[1, 1, 5].isnan().all()) and bool(out[0, 2, 0].isnan().all())
    rest = torch.ones(2, n, 8, dtype=torch.bool, device="cuda")
    rest[1, 1, 5] = rest[0, 2, 0] = False
    assert torch.equal(out[rest], clean[rest])


@pytest.mark.parametrize("room", [None, 2000])
@pytest.mark.parametrize("n", [1, 40])
def test_attend_page_outside_the_pool(n, room):
    """Its tokens are not seen; rows that see nothing else are no number."""
    p = Pool((8, 2, 128), 16, [n + 40, n + 1, 7], [n, n, 0], seed=n, width=room)
    for b, i, to in ((0, 1, 1 << 20), (1, 0, -1)):
        p.table_h[b][i] = to
    p.table.copy_(dev(p.table_h))
    out = p.attend()
    assert p.ops.errors(stream()) == ERR_PAGE and p.ops.errors(stream()) == 0
    # request 0 without slots 16 .. 31: the same as a row whose second page is left out
    table = [[x for i, x in enumerate(p.table_h[0]) if i != 1] + [-1], p.table_h[1], p.table_h[2]]
    q = Pool((8, 2, 128), 16, [n + 40, n + 1, 7], [n, n, 0], seed=n, width=room)
    q.table.copy_(dev(table))
    q.lens.copy_(dev([n + 24, 0, 7]))
    q.new.copy_(dev([n, 0, 0]))
    want = q.attend()[0]
    size = want.abs().amax()
    assert bool(((out[0] - want).abs() <= 64 * U * size).all())  # (sums of the same terms in another order)
    seen = [t for t in range(n) if 1 + t >= 16]
    assert bool(out[1, [t for t in range(n) if t not in seen]].isnan().all())
    assert bool((out[2] == 7.0).all())


@pytest.mark.parametrize("bad", [dict(lens=[-1, 9]), dict(lens=[1000, 9]), dict(new=[6, 2]), dict(new=[-1, 2]), dict(lens=[1, 9])])
def test_attend_request_out_of_range_is_left_out(bad):
    p = Pool((8, 2, 64), 16, [9, 9], [2, 2], seed=5)
    want = p.attend().clone()
    assert p.ops.errors(stream()) == 0
    p.lens.copy_(dev(bad.get("lens", [9, 9])))
    p.new.copy_(dev(bad.get("new", [2, 2])))
    p.out.fill_(7.0)
    out = p.attend()
    assert bool((out[0] == 7.0).all()) and torch.equal(out[1], want[1])
    assert p.ops.errors(stream()) == ERR_LENS


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("scale", [2.0**-20, 2.0**-12, 2.0**4, 2040.0])
def test_attend_scales(scale, n):
    """Values as small and as large as 4 bits hold; the scores' scale undone by the queries."""
    p = Pool((8, 2, 128), 32, [77, 43], [n, n], seed=6, width=1000)
    pool = p.pool_h.copy()
    d = np.sign(np.random.default_rng(1).standard_normal(pool[:, :, 32 * 128 :].shape[:-1] + (2 * 32 * 4,))) * scale
    pool[:, :, 32 * 128 :] = d.astype(np.float16).view(np.uint8).reshape(pool.shape[0], 2, -1)
    p.pool.copy_(torch.from_numpy(pool))
    p.q *= 0.1 / scale
    p.check_all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("room", [None, 4000])
@pytest.mark.parametrize("n", [1, 5, 40])
@pytest.mark.parametrize("gap", [8, 12, 16, 20, 24])
def test_attend_sink(gap, n, room, hd):
    """A first key that outweighs all others together and whose value is 0: the output is the others', whose weights are far
    below the row's largest.  Beside the bounds of sums in f32, a weight is held to 2^-22 of itself or 2^-39 of the largest of
    its row (two f16 parts, the largest at 2^14 or above, half a step of the least f16 numbers 2^-25)."""
    p = Pool((8, 2, hd), 16, [n + 1000, n + 90, n + 1], [n] * 3, seed=gap + n, width=room)
    sign = np.where(np.random.default_rng(gap).random(hd) < 0.5, -7, 7)
    pool = p.pool_h.copy()
    for row in p.table_h:
        for g in range(2):
            p.lay.write(pool[row[0], g], 0, (sign + 8, np.ones(hd // 32)), (np.full(hd, 8), np.zeros(hd // 32)))
    p.pool.copy_(torch.from_numpy(pool))
    p.q.mul_(0.1).add_(torch.as_tensor(sign, device="cuda") * (gap / 49 / math.sqrt(hd)))
    out = p.attend()
    k, v = p.dense()
    ref, tol = kv_util.attend(p.q, k, v, p.lens_h, p.new_h)[:2]
    for b in range(3):
        upto = v[b].abs().cumsum(1)[:, p.lens_h[b] - n : p.lens_h[b]]  # [G][n][hd]: of the values that a token sees
        tol[b] += 2.0**-39 * upto.transpose(0, 1).repeat_interleave(4, 1)
    p.check(out, (ref, tol))
    assert p.ops.errors(stream()) == 0


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("room", [None, 4000])
@pytest.mark.parametrize("n", [1, 5, 40])
@pytest.mark.parametrize("below", [False, True])  # 0: all scores are negative
def test_attend_large_scores(below, n, room, hd):
    """Scores of 2^12 to 2^40 (where f32 has whole numbers, then every 2nd, 4th ..): the largest, a sixth or more above the others,
    takes all of the weight, and its value comes out."""
    p = Pool((8, 2, hd), 16, [n + 1000, n + 90, n + 6], [n] * 3, seed=n, width=room)
    r = np.random.default_rng(n)
    pool, best = p.pool_h.copy(), 5
    code = np.full(hd, 8)
    zero = code, np.zeros(hd // 32)
    for b, row in enumerate(p.table_h):
        for s in range(p.lens_h[b]):
            for g in range(2):
                part, lay = pool[row[s // 16], g], p.lay
                at, shift = lay.key[0][s % 16, :32], lay.key[1][s % 16, :32]  # the first group: one dim, the other groups' scales are 0
                part[lay.key_scale[s % 16][:, None] + np.arange(2)] = 0
                part[lay.key_scale[s % 16, 0] + np.arange(2)] = np.array([1.0], np.float16).view(np.uint8)
                c = (7 if s == best else r.integers(-8, 7)) if not below else (-1 if s == best else -r.integers(2, 9))
                part[at] = 0x88
                part[at[0]] = (0x88 & ~(15 << int(shift[0])) & 255) | int(c + 8) << int(shift[0])
    p.pool.copy_(torch.from_numpy(pool))
    v = p.dense()[1]
    want = v[:, :, best].repeat_interleave(4, 1)[:, None].expand(p.out.shape)
    mantissa = 1 + torch.rand(p.q.shape[:3], generator=gen(n), device="cuda")
    for e in range(12, 40):
        p.q.zero_()
        p.q[..., 0] = mantissa * 2.0**e
        p.out.fill_(7.0)
        out = p.attend()
        far = (out.double() - want).abs()
        assert bool((far <= 4 * U * want.abs()).all()), (e, far.max().item())
    assert p.ops.errors(stream()) == 0


def test_attend_offsets_beyond_32_bits():
    """Pages that lie more than 4 GiB into the pool."""
    page, hd, G = 128, 128, 8
    lay = pages_util.Layout(page, hd)
    count = (5 << 30) // (G * lay.part)
    ops = PagedKv(32, G, hd, page, count, 4, max_requests=2, max_tokens=8)
    small = Pool((32, G, hd), page, [300, 200], [1, 1], seed=8)
    pool = torch.zeros(count, G, lay.part, dtype=torch.uint8, device="cuda")
    table = [[x + count - small.pages if x >= 0 else -1 for x in row] for row in small.table_h]
    pool[count - small.pages :] = small.pool
    t = dev(table)
    ops.attend(ops.view(ptr(pool), ptr(t), ptr(small.lens), 2, new_lens=ptr(small.new)), ptr(small.q), 1, ptr(small.out), stream=stream())
    torch.cuda.synchronize()
    small.check(small.out)
    refs = torch.zeros(count, dtype=torch.int32, device="cuda")
    refs[t[t >= 0].long()] = 1
    used = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.compact(ops.view(ptr(pool), ptr(t), ptr(small.lens), 2), ptr(refs), ptr(refs), ptr(t), ptr(used), stream=stream())
    small.out.fill_(7.0)
    ops.attend(ops.view(ptr(pool), ptr(t), ptr(small.lens), 2, new_lens=ptr(small.new)), ptr(small.q), 1, ptr(small.out), stream=stream())
    torch.cuda.synchronize()
    small.check(small.out)
    assert int(used) == int(refs.sum()) == 5 and bool((refs[:5] == 1).all()) and int(t.max()) == 4
    assert ops.errors(stream()) == 0


@pytest.mark.parametrize("shape,n", [((64, 1, 64), 2), ((4, 4, 128), 100), ((64, 1, 64), 1), ((8, 1, 128), 3)])
def test_attend_most_states(shape, n):
    """Tables of 2^20 slots, runs far shorter: as many splits of a row tile, and states, as a call has."""
    Pool(shape, 128, [3000 + n], [n], seed=n, width=8192).check_all()


def test_memory_of_a_handle():
    """What a handle keeps at head dim 128: no more attention states than calls leave."""
    torch.cuda.synchronize()
    PagedKv(8, 2, 128, 16, 10, 4, max_requests=1).close()  # (what the runtime takes with the first)
    before = torch.cuda.mem_get_info()[0]
    ops = PagedKv(8, 2, 128, 16, 10, 4, max_requests=1)
    taken = before - torch.cuda.mem_get_info()[0]
    ops.close()
    assert taken <= 40 << 20, taken  # 4096 states of 16 rows of 130 numbers are 32.5 MiB, the rest below 10 KB in arrays of their own


def test_attend_most_tokens():
    """The most tokens of a call, 4 M packed rows; a few of them against 64 bits."""
    n, page, hd = 32768, 128, 64
    lens = [n + 5, n + 1]
    p = Pool((64, 1, hd), page, lens, [n, n], seed=12)
    p.attend()
    k, v = p.dense()
    for b in range(2):
        for t in (0, 1, 16383, 16384, n - 1):
            seen = lens[b] - n + t + 1
            want, tol = kv_util.attend(p.q[b : b + 1, t : t + 1], k[b : b + 1], v[b : b + 1], [seen], [1])[:2]
            assert bool(((p.out[b : b + 1, t : t + 1].double() - want).abs() <= tol).all()), (b, t)
    assert p.ops.errors(stream()) == 0 and not bool((p.out == 7.0).all(-1).any())


# --------------------------------------------------------------------------
# append
# --------------------------------------------------------------------------
class Append:
    def __init__(self, shape, page, lens, new, dims=0, half=False, scaling="none", factor=1.0, norms=True, spread=3.0, seed=0, held=True, far=60000):
        self.pool = Pool(shape, page, lens, new, seed=seed, rope_half=half, eps=1e-6, rope_dims=dims,
                         **(dict(zip(("rope_freq", "rope_gain"), rope_frequencies(dims or shape[2], 1.0e6, scaling, factor))) if scaling != "none" else {}))
        p = self.pool
        g = gen(seed + 1)
        self.dims, self.half = dims or p.hd, half
        self.freq, self.mult = rope_frequencies(self.dims, 1.0e6, scaling, factor)
        self.qkv = normal(g, p.R, p.n, p.H + 2 * p.G, p.hd, spread=spread)
        self.qn = normal(g, p.hd, spread=0.2) + 1 if norms else None
        self.kn = normal(g, p.hd, spread=0.2) + 1 if norms else None
        self.pos = torch.randint(0, far, (p.R, p.n), generator=g, device="cuda", dtype=torch.int32)
        self.q = torch.full((p.R, p.n, p.H, p.hd), 7.0, device="cuda")
        self.k_held = torch.full((p.R, p.n, p.G, p.hd), 7.0, device="cuda") if held else None
        self.v_held = torch.full((p.R, p.n, p.G, p.hd), 7.0, device="cuda") if held else None

    def run(self):
        p = self.pool
        p.ops.append(p.view(), ptr(self.qkv), p.n, ptr(self.pos), ptr(self.q), q_norm=ptr(self.qn), k_norm=ptr(self.kn), k_held=ptr(self.k_held),
                     v_held=ptr(self.v_held), stream=stream())
        torch.cuda.synchronize()

    def check(self):
        p = self.pool
        x = self.qkv.double().cpu()
        pos = self.pos.cpu()
        eps = float(torch.tensor(1e-6))
        norm = lambda g: None if g is None else g.cpu()  # noqa: E731
        q = pages_util.rotated(x[:, :, : p.H], pos, norm(self.qn), self.dims, self.half, self.freq, self.mult, eps)
        k = pages_util.rotated(x[:, :, p.H : p.H + p.G], pos, norm(self.kn), self.dims, self.half, self.freq, self.mult, eps)
        v = x[:, :, p.H + p.G :]
        pool = p.pool_h.copy()
        want_k, want_v = torch.full((p.R, p.n, p.G, p.hd), 7.0), torch.full((p.R, p.n, p.G, p.hd), 7.0)
        for b in range(p.R):
            for t in range(p.new_h[b]):
                slot = p.lens_h[b] - p.new_h[b] + t
                for g in range(p.G):
                    key, val = pages_util.quantised(k[b, t, g].numpy()), pages_util.quantised(v[b, t, g].numpy())
                    p.lay.write(pool[p.table_h[b][slot // p.page], g], slot % p.page, key[:2], val[:2])
                    want_k[b, t, g], want_v[b, t, g] = torch.from_numpy(key[2]), torch.from_numpy(val[2])
        live = torch.arange(p.n)[None] < torch.tensor(p.new_h)[:, None]
        got = self.q.cpu()
        assert bool((got[~live] == 7.0).all())
        # one rounding to f32, and 2^-32 of the head for norm, angle and rotation in 64 bits
        far = (got.double() - q).abs()
        assert bool((far <= U * q.abs() + 2.0**-32 * q.norm(dim=-1, keepdim=True))[live].all())
        if self.k_held is not None:
            assert torch.equal(self.k_held.cpu(), want_k) and torch.equal(self.v_held.cpu(), want_v)
        assert np.array_equal(p.pool.cpu().numpy(), pool)
        assert p.ops.errors(stream()) == 0


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_append(shape, page):
    a = Append(SHAPES[shape], page, [1, 17, 16, 40], [1, 3, 0, 2], seed=page)
    a.run()
    a.check()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("dims", [16, 32, 64, 128])
@pytest.mark.parametrize("scaling", ["none", "linear", "stretch", "parts"])
def test_append_rotations(dims, half, scaling):
    a = Append((8, 2, 128), 32, [9, 50], [4, 2], dims=dims, half=half, scaling=scaling, factor=4.0, seed=dims)
    a.run()
    a.check()
    if dims <= 64:
        a = Append((4, 4, 64), 16, [9], [3], dims=dims, half=half, scaling=scaling, factor=8.0, seed=dims)
        a.run()
        a.check()


@pytest.mark.parametrize("dims", [2, 6, 30, 62])
def test_append_few_dims(dims):
    a = Append((8, 2, 64), 16, [9, 30], [4, 1], dims=dims, seed=dims)
    a.run()
    a.check()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("dims,hd", [(16, 64), (32, 128), (64, 128), (128, 128)])
def test_append_infinities_beside_dims_that_do_not_turn(dims, hd, half):
    """The rest of a head is as it is, whatever stands in the other dims and in itself."""
    a = Append((4, 2, hd), 16, [5, 30], [5, 2], dims=dims, half=half, norms=False, seed=dims)
    for t in range(2):
        a.qkv[:, t, 0, hd - 2 :] = torch.tensor([[math.inf, 1.5], [-2.0, -math.inf]], device="cuda")[t]
        a.qkv[:, t, 1, hd - 8 :: 3] = math.nan
        a.qkv[:, t, 2, min(dims, hd - 1)] = -math.inf
        a.qkv[:, t, 3, t] = math.inf
    a.run()
    x = a.qkv.cpu()[:, :, :4]
    want = pages_util.rotated(x, a.pos.cpu(), None, dims, half, a.freq, a.mult, 0.0).float()
    for b, new in enumerate(a.pool.new_h):
        got = a.q[b, :new].cpu()
        assert np.array_equal(got[..., dims:].numpy(), x[b, :new, :, dims:].numpy(), equal_nan=True)
        assert torch.equal(got.isnan(), want[b, :new].isnan()) and torch.equal(got.isinf(), want[b, :new].isinf())
    assert a.pool.ops.errors(stream()) == 0  # (no key and no value of no number)


def test_append_without_norms_or_held():
    a = Append((8, 2, 128), 32, [9, 70], [9, 40], norms=False, held=False, seed=3)
    a.run()
    a.check()


@pytest.mark.parametrize("n", [2, 3, 4, 5, 8, 31, 70])
def test_append_turns(n):
    """From one token to several pages, from any slot on."""
    a = Append((8, 2, 128), 16, [n, n + 1, n + 2, n + 7, n + 30], [n, n, n - 1, n, max(1, n // 2)], seed=n)
    a.run()
    a.check()


def test_append_far_positions():
    a = Append((8, 2, 128), 16, [3, 30], [3, 2], seed=1, far=(1 << 31) - 1)
    a.run()
    p = a.pool
    q = pages_util.rotated(a.qkv.double().cpu()[:, :, : p.H], a.pos.cpu(), a.qn.cpu(), 128, False, a.freq, a.mult, 1e-6)
    live = torch.arange(p.n)[None] < torch.tensor(p.new_h)[:, None]
    # angles of 2^31 radians are exact to 2^-22 either way
    assert bool(((a.q.cpu().double() - q).abs() <= 2.0**-20 * q.norm(dim=-1, keepdim=True))[live].all())


def _values(x):
    """Appends x [tokens][32] as the first group of values of a one-head cache; what is held of it, and the errors."""
    n = x.shape[0]
    a = Append((1, 1, 64), 16, [n], [n], seed=2, norms=False)
    a.qkv[0, :, 2, :32] = torch.as_tensor(x, dtype=torch.float32).cuda()
    a.run()
    return a, a.v_held[0, :, 0, :32].cpu().double().numpy()


def test_append_equals_and_ties():
    """The first of equals gives the sign; halves go to even codes; zeros."""
    up, down = np.zeros(32), np.zeros(32)
    up[3], up[9] = 8.0, -8.0
    down[3], down[9] = -8.0, 8.0
    half = np.array([-8.0] + [i / 2 for i in range(-16, 15)])
    near = np.array([-8.0] + [np.nextafter(np.float32(i / 2), np.float32(9 if i % 4 else -9)) for i in range(-16, 15)])
    _, held = _values(np.stack([up, down, half, near, np.zeros(32), -half * 3]))
    for got, x in zip(held, [up, down, half, near, np.zeros(32), -half * 3]):
        assert np.array_equal(got, pages_util.quantised(x.astype(np.float32))[2])
    assert held[0, 3] == 8.0 and held[0, 9] == -7.0 and held[1, 3] == -8.0 and held[1, 9] == 7.0


def test_append_small_and_large():
    r = np.random.default_rng(5)
    x = (r.standard_normal((40, 32)) * 2.0 ** r.integers(-30, 12, (40, 1))).astype(np.float32)
    x[0] *= 16383.0 / np.abs(x[0]).max()
    x = np.clip(x, -16383, 16383)
    a, held = _values(x)
    for got, y in zip(held, x):
        assert np.array_equal(got, pages_util.quantised(y)[2])
    assert a.pool.ops.errors(stream()) == 0


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 16384.0, -1e30])
def test_append_beyond_the_range(bad):
    x = np.ones((3, 32))
    x[1, 20] = bad
    a, held = _values(x)
    assert np.isnan(held[1]).all() and (held[[0, 2]] == pages_util.quantised(x[0])[2]).all()
    assert a.pool.ops.errors(stream()) == ERR_RANGE
    k, v = a.pool.dense()
    assert bool(v[0, 0, 1, :32].isnan().all()) and bool(torch.isfinite(v[0, 0, 1, 32:64]).all()) and bool(torch.isfinite(v[0, 0, [0, 2]]).all())


def test_append_rows_of_no_token_may_hold_anything():
    a = Append((8, 2, 128), 16, [20, 20], [2, 5], seed=4)
    a.qkv[0, 2:] = math.nan
    a.pos[0, 2:] = -7
    a.run()
    a.qkv[0, 2:] = 0
    a.pos[0, 2:] = 0
    a.check()


def test_append_what_is_left_out():
    a = Append((8, 2, 128), 16, [20, 20, 20], [3, 3, 3], seed=6)
    p = a.pool
    clean = Append((8, 2, 128), 16, [20, 20, 20], [3, 3, 3], seed=6)
    clean.run()
    a.pos[0, 1] = -1
    p.lens.copy_(dev([20, 2, 20]))
    table = [list(r) for r in p.table_h]
    table[2][1] = p.pages
    p.table.copy_(dev(table))
    a.run()
    assert p.ops.errors(stream()) == ERR_POSITION | ERR_LENS | ERR_PAGE
    assert bool((a.q[0, 1] == 7.0).all()) and torch.equal(a.q[0, [0, 2]], clean.q[0, [0, 2]])
    assert bool((a.q[1] == 7.0).all()) and torch.equal(a.q[2], clean.q[2])  # (a query needs no page)
    got, want, old = p.pool.cpu().numpy(), clean.pool.pool.cpu().numpy(), p.pool_h
    lay, at = p.lay, p.table_h[0][1]
    for s in range(16):
        exp = want if s in (1, 3) else old  # slots 17 .. 19 of request 0, the middle one left out
        assert np.array_equal(got[at][:, lay.key[0][s]], exp[at][:, lay.key[0][s]]) and np.array_equal(got[at][:, lay.value_scale[s]], exp[at][:, lay.value_scale[s]])
    others = [x for x in range(p.pages) if x != at]
    assert np.array_equal(got[others], old[others])


# --------------------------------------------------------------------------
# update, compact
# --------------------------------------------------------------------------
class Book:
    """Rows of pages in three layers on the device, and their model in Python."""

    def __init__(self, rows, width, pages, page=16, layers=3, seed=0):
        self.rows, self.width, self.pages, self.page, self.layers = rows, width, pages, page, layers
        self.ops = PagedKv(4, 1, 64, page, pages, width, max_requests=rows, max_tokens=64)
        self.table, self.lens, self.refs = [[-1] * width for _ in range(rows)], [0] * rows, [0] * pages
        r = np.random.default_rng(seed)
        self.pool = r.integers(-(1 << 31), 1 << 31, (layers, pages, self.ops.page_bytes // 4), dtype=np.int64).astype(np.int32)
        self.d = {k: dev(getattr(self, k)) for k in ("table", "lens", "refs")}
        self.d_pool = torch.from_numpy(self.pool).cuda()

    def view(self):
        return self.ops.view(ptr(self.d_pool), ptr(self.d["table"]), ptr(self.d["lens"]), self.rows)

    def outs(self, in_place):
        return {k: (v if in_place else torch.full_like(v, 99)) for k, v in self.d.items()}

    def update(self, source=None, keep=None, add=None, in_place=True, errors=0):
        n, out = self.rows, self.outs(in_place)
        args = {k: dev(v) for k, v in (("source", source), ("keep", keep), ("add", add)) if v is not None}
        before = {k: v.clone() for k, v in self.d.items()}
        self.ops.update(self.view(), ptr(self.d["refs"]), ptr(out["refs"]), ptr(out["table"]), ptr(out["lens"]), layers=self.layers, stream=stream(),
                        **{k: ptr(v) for k, v in args.items()})
        torch.cuda.synchronize()
        if not in_place:
            assert all(torch.equal(self.d[k], before[k]) for k in before)
        self.d = out
        res = pages_util.update(self.table, self.lens, self.refs, list(range(n)) if source is None else source, [1 << 30] * n if keep is None else keep,
                                [0] * n if add is None else add, self.page, self.width)
        assert self.ops.errors(stream()) == errors and (res is None) == (errors != 0)
        if res:
            self.table, self.lens, self.refs, copies = res
            old = self.pool.copy()
            for to, at in copies.items():
                self.pool[:, to] = old[:, at]
        self.check()

    def compact(self, in_place=True):
        out = self.outs(in_place)
        out["lens"] = self.d["lens"]
        if not in_place:
            out["table"] = self.d["table"].clone()
        used, moved = dev([-1]), torch.full((self.pages,), 99, dtype=torch.int32, device="cuda")
        self.ops.compact(self.view(), ptr(self.d["refs"]), ptr(out["refs"]), ptr(out["table"]), ptr(used), moved_to=ptr(moved), layers=self.layers, stream=stream())
        torch.cuda.synchronize()
        self.d = out
        refs = self.refs
        self.table, self.refs, to, n = pages_util.compact(self.table, self.lens, self.refs, self.page)
        for a, b in to.items():
            self.pool[:, b] = self.pool[:, a]
        assert int(used) == n and moved.tolist() == [(to.get(p, p) if r > 0 else -1) for p, r in enumerate(refs)]
        assert self.ops.errors(stream()) == 0
        self.check()

    def check(self):
        assert self.d["lens"].tolist() == self.lens
        assert self.d["table"].tolist() == self.table
        assert self.d["refs"].tolist() == self.refs
        assert np.array_equal(self.d_pool.cpu().numpy(), self.pool)


@pytest.mark.parametrize("in_place", [True, False])
def test_update_a_session(in_place):
    k = Book(6, 8, 40)
    k.update(add=[40, 0, 0, 0, 0, 0], in_place=in_place)  # a prompt
    k.update(source=[0, 0, 0, 0, -1, 5], add=[0, 1, 1, 1, 0, 0], in_place=in_place)  # three fork it and grow
    k.update(add=[1, 1, 1, 1, 0, 0], in_place=in_place)  # the last holder keeps the page
    k.update(keep=[0, 100, 20, 100, 0, 0], in_place=in_place)  # one ends, one is cut back
    k.update(source=[2, 3, 1, 1, 1, 1], add=[3, 0, 17, 1, 0, 128 - 42], in_place=in_place)  # beams sorted anew
    k.update(source=[-1] * 6, in_place=in_place)
    assert sum(k.refs) == 0


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("pages", [7, 20000])  # spare ones: few, and so many that the counts do not fit a block's LDS
@pytest.mark.parametrize("seed", range(6))
def test_update_and_compact_at_random(seed, pages, in_place):
    g = random.Random(seed)
    rows, page = g.choice([1, 2, 5, 17, 64]), g.choice([16, 32, 64, 128]) if pages < 100 else 16
    width = g.choice([1, 3, 12])
    k = Book(rows, width, rows * width + pages, page=page, layers=g.choice([1, 2]) if pages < 100 else 1, seed=seed)
    for i in range(25):
        if i % 6 == 5:
            k.compact(in_place)
            continue
        source = [g.randrange(-1, rows) if g.random() < 0.3 else b for b in range(rows)]
        keep = [g.choice([0, page, page + 1, g.randint(0, width * page)]) if g.random() < 0.3 else 1 << 30 for _ in range(rows)]
        left = [width * page - (0 if s < 0 else min(n, k.lens[s])) for s, n in zip(source, keep)]
        add = [g.choice([0, 1, 1, m, g.randint(0, m), min(m, page)]) if m else 0 for m in left]
        add = [min(a, m) for a, m in zip(add, left)]
        k.update(source, keep, add, in_place)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("seed", range(2))
def test_update_and_compact_counts_beyond_lds(seed, in_place):
    test_update_and_compact_at_random(seed, 40000, in_place)


@pytest.mark.parametrize("in_place", [True, False])
def test_update_refused(in_place):
    """Whatever is wrong: nothing changes."""
    k = Book(3, 4, 9)
    k.update(add=[40, 20, 0])
    k.update(add=[0, 0, 65], errors=ERR_LENS, in_place=in_place)
    k.update(add=[25, 0, 0], errors=ERR_LENS, in_place=in_place)
    k.update(add=[0, -1, 0], errors=ERR_LENS, in_place=in_place)
    k.update(keep=[0, -1, 0], errors=ERR_LENS, in_place=in_place)
    k.update(source=[0, 3, 0], errors=ERR_LENS, in_place=in_place)
    k.update(source=[0, -2, 0], errors=ERR_LENS, in_place=in_place)
    k.update(add=[8, 28, 64], errors=ERR_FULL, in_place=in_place)  # 3 + 2 in use; 0 + 1 + 4 more of 4 free
    k.update(source=[0, 0, 0], add=[2, 2, 60 - 40], errors=0, in_place=in_place)
    lens = k.lens
    k.lens = [lens[0], 65, lens[2]]
    k.d["lens"].copy_(dev(k.lens))
    k.update(errors=ERR_LENS, in_place=in_place)
    k.lens = lens
    k.d["lens"].copy_(dev(lens))
    was, k.table[1][0] = k.table[1][0], 9
    k.d["table"].copy_(dev(k.table))
    k.update(errors=ERR_PAGE, in_place=in_place)
    k.table[1][0] = was
    k.d["table"].copy_(dev(k.table))
    full, k.refs[was] = k.refs[was], 1
    assert full > 1
    k.d["refs"].copy_(dev(k.refs))
    k.update(source=[-1, -1, -1], errors=ERR_REFS, in_place=in_place)
    k.refs[was], k.refs[8] = 0, 0
    k.d["refs"].copy_(dev(k.refs))
    k.update(add=[1, 0, 0], errors=ERR_REFS, in_place=in_place)  # a page that a row keeps, counted by none
    k.refs[was], k.refs[8] = full, -1
    k.d["refs"].copy_(dev(k.refs))
    k.update(errors=ERR_REFS, in_place=in_place)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("pages", [12, 20000, 40000])  # all in a block's LDS, the counts alone, nothing
def test_update_counts_below_the_rows(pages, in_place):
    """A page counted by fewer than the rows that hold it: no row takes it for its own, whatever the rows become."""
    k = Book(4, 4, pages, layers=1)
    k.update(add=[20, 0, 37, 0])
    k.update(source=[0, 0, 2, 0])  # rows 0, 1 and 3 hold two pages in common, the second not full
    first, second = k.table[0][:2]
    assert k.refs[first] == k.refs[second] == 3
    for page, refs in ((second, 2), (second, 1), (first, 2)):
        short = list(k.refs)
        short[page] = refs
        for args in (dict(add=[1, 1, 0, 1]), dict(add=[1, 0, 0, 0]), dict(keep=[18, 99, 99, 99], add=[1, 0, 0, 0]), dict(), dict(add=[0, 0, 1, 0]),
                     dict(source=[0, 1, 0, -1], add=[1, 1, 1, 0]), dict(source=[-1, 1, 2, 3]), dict(source=[0, -1, 2, -1], add=[1, 0, 0, 0])):
            d, args = dict(k.d, refs=dev(short)), {x: dev(y) for x, y in args.items()}
            before = {x: y.clone() for x, y in d.items()}
            out = {x: (y if in_place else torch.full_like(y, 99)) for x, y in d.items()}
            k.ops.update(k.ops.view(ptr(k.d_pool), ptr(d["table"]), ptr(d["lens"]), 4), ptr(d["refs"]), ptr(out["refs"]), ptr(out["table"]), ptr(out["lens"]),
                         stream=stream(), **{x: ptr(y) for x, y in args.items()})
            torch.cuda.synchronize()
            assert k.ops.errors(stream()) == ERR_REFS, (page, refs, args)
            assert all(torch.equal(out[x], before[x]) and torch.equal(d[x], before[x]) for x in d)
            k.check()
    k.update(add=[1, 1, 0, 1], in_place=in_place)


@pytest.mark.parametrize("in_place", [True, False])
def test_compact_counts_below_the_rows(in_place):
    """Compact looks for pages that a row holds and no one counts; a count that is only too low moves with its page."""
    k = Book(3, 4, 12)
    k.update(add=[40, 20, 20])
    k.update(source=[-1, 1, 1])
    page = k.table[1][1]
    assert page > 1 and k.refs[page] == 2
    k.refs[page] = 1
    k.d["refs"].copy_(dev(k.refs))
    k.compact(in_place)
    assert k.refs[:3] == [2, 1, 0]


def test_update_full_to_the_last_page():
    k = Book(2, 8, 9)
    k.update(add=[128, 16, ])
    k.update(add=[0, 1], errors=ERR_FULL)
    k.update(keep=[112, 16], add=[0, 1])


def test_compact_refused():
    k = Book(2, 4, 12)
    k.update(add=[40, 40])
    k.update(keep=[0, 40])
    for what, value, bits in (("lens", [0, 65], ERR_LENS), ("table", [[-1] * 4, [3, 12, 5, -1]], ERR_PAGE), ("refs", [0, 0, 0, 1, 0, 1] + [0] * 6, ERR_REFS),
                              ("refs", [-1, 0, 0, 1, 1, 1] + [0] * 6, ERR_REFS)):
        for in_place in (True, False):
            d = dict(k.d, **{what: dev(value)})
            before, pool = {x: y.clone() for x, y in d.items()}, k.d_pool.clone()
            out = {x: (y if in_place else torch.full_like(y, 99)) for x, y in d.items()}
            used = dev([-1])
            k.ops.compact(k.ops.view(ptr(k.d_pool), ptr(d["table"]), ptr(d["lens"]), 2), ptr(d["refs"]), ptr(out["refs"]), ptr(out["table"]), ptr(used),
                          layers=3, stream=stream())
            assert k.ops.errors(stream()) == bits
            assert torch.equal(out["table"], before["table"]) and torch.equal(out["refs"], before["refs"]) and torch.equal(k.d_pool, pool)


def test_rows_of_large_tables():
    k = Book(64, 300, 20000, page=16, layers=1)
    g = random.Random(5)
    k.update(add=[g.randint(0, 4800) for _ in range(64)])
    k.update(source=[g.randrange(64) for _ in range(64)], keep=[g.randint(0, 4800) for _ in range(64)])
    k.update(add=[min(g.randint(0, 50), 4800 - n) for n in k.lens], in_place=False)
    k.update(keep=[0 if b % 2 else 1 << 30 for b in range(64)])
    k.compact()
    k.compact(in_place=False)


@pytest.mark.parametrize("in_place", [True, False])
def test_update_most_rows(in_place):
    """256 rows: all fork one, grow into its last page, and are sorted anew."""
    k = Book(256, 3, 700, page=16, layers=1)
    k.update(add=[20] + [0] * 255, in_place=in_place)
    k.update(source=[0] * 256, add=[b % 3 for b in range(256)], in_place=in_place)
    k.update(source=list(range(255, -1, -1)), add=[1] * 256, in_place=in_place)
    k.update(source=[b // 2 for b in range(256)], keep=[21 + b % 3 for b in range(256)], in_place=in_place)
    k.compact(in_place)


@pytest.mark.parametrize("in_place", [True, False])
def test_update_what_else_holds_pages(in_place):
    """Counts that no row of the table stands for: a page with one is neither free nor any row's alone."""
    k = Book(3, 4, 12)
    k.update(add=[20, 16, 5], in_place=in_place)
    for p in (k.table[0][1], k.table[2][0], 9):
        k.refs[p] += 1
    k.d["refs"].copy_(dev(k.refs))
    k.update(add=[1, 1, 0], in_place=in_place)  # row 0 grows into a copy
    k.update(keep=[0, 17, 0], in_place=in_place)
    assert [p for p, n in enumerate(k.refs) if n] and k.refs[9] == 1
    k.update(add=[64, 0, 0], in_place=in_place)


@pytest.mark.parametrize("in_place", [True, False])
def test_largest_pool(in_place):
    """2^20 pages, many of them held by others: the rows grow into free ones, then the pool is compacted."""
    pages, page, width, rows = 1 << 20, 16, 40, 3
    ops = PagedKv(4, 1, 64, page, pages, width, max_requests=rows, max_tokens=64)
    pool = torch.zeros(pages, ops.page_bytes // 4, dtype=torch.int32, device="cuda")
    pool[:, 0] = pool[:, -1] = torch.arange(pages, device="cuda")
    r = np.random.default_rng(3)
    held = np.where(r.random(pages) < 0.999, r.integers(1, 4, pages), 0)
    held[-50000:] = 0
    table, lens, refs = [[-1] * width for _ in range(rows)], [0] * rows, held.tolist()
    d = [dev(x) for x in (table, lens, refs)]
    for source, keep, add in (([0, 1, 2], [0, 0, 0], [600, 333, 0]), ([0, 0, 1], [599, 100, 333], [41, 1, 64])):
        out = d if in_place else [torch.full_like(x, 99) for x in d]
        args = [dev(x) for x in (source, keep, add)]
        ops.update(ops.view(ptr(pool), ptr(d[0]), ptr(d[1]), rows), ptr(d[2]), ptr(out[2]), ptr(out[0]), ptr(out[1]), source=ptr(args[0]), keep=ptr(args[1]), add=ptr(args[2]), stream=stream())
        table, lens, refs, copies = pages_util.update(table, lens, refs, source, keep, add, page, width)
        d = out
        assert [x.tolist() for x in d] == [table, lens, refs]
        for to, at in copies.items():
            assert pool[to, 0] == at and pool[to, -1] == at
            pool[to, 0] = pool[to, -1] = to
    used, moved = dev([-1]), torch.full((pages,), 99, dtype=torch.int32, device="cuda")
    out = d if in_place else [d[0].clone(), d[1], torch.full_like(d[2], 99)]
    ops.compact(ops.view(ptr(pool), ptr(d[0]), ptr(d[1]), rows), ptr(d[2]), ptr(out[2]), ptr(out[0]), ptr(used), moved_to=ptr(moved), stream=stream())
    was = np.array(refs)
    table, refs, to, n = pages_util.compact(table, lens, refs, page)
    assert ops.errors(stream()) == 0 and len(to) > 0 and int(used) == n
    assert out[0].tolist() == table and out[2].tolist() == refs
    want = np.where(was > 0, np.arange(pages), -1)
    want[list(to)] = list(to.values())
    assert np.array_equal(moved.cpu().numpy(), want)
    at = moved[moved >= 0].long()
    names = torch.arange(pages, device="cuda")[moved >= 0].int()
    assert torch.equal(pool[at, 0], names) and torch.equal(pool[at, -1], names)


def test_layers_apart():
    k = Book(3, 4, 8, layers=2)
    gap = torch.full((2, 8 * k.ops.page_bytes + 64), 3, dtype=torch.uint8, device="cuda")
    k.update(add=[20, 0, 0])
    bytes_ = k.d_pool.view(torch.uint8).view(2, -1)
    gap[:, : bytes_.shape[1]] = bytes_
    args = [dev([0, 0, 0]), dev([1, 1, 1])]
    want = pages_util.update(k.table, k.lens, k.refs, [0, 0, 0], [1 << 30] * 3, [1, 1, 1], 16, 4)
    k.ops.update(k.ops.view(ptr(gap), ptr(k.d["table"]), ptr(k.d["lens"]), 3), ptr(k.d["refs"]), ptr(k.d["refs"]), ptr(k.d["table"]), ptr(k.d["lens"]),
                 source=ptr(args[0]), add=ptr(args[1]), layers=2, layer_stride=gap.shape[1], stream=stream())
    torch.cuda.synchronize()
    assert k.d["table"].tolist() == want[0] and len(want[3]) == 2
    for to, at in want[3].items():
        k.pool[:, to] = k.pool[:, at]
    assert np.array_equal(gap[:, : bytes_.shape[1]].cpu().numpy().view(np.int32).reshape(k.pool.shape), k.pool)
    assert bool((gap[:, bytes_.shape[1] :] == 3).all())


# --------------------------------------------------------------------------
# together
# --------------------------------------------------------------------------
class Sessions:
    """What a server runs per step, with one layer: rows made anew, tokens appended, attention."""

    def __init__(self, rows=4, page=16, width=12, pages=60, shape=(8, 2, 64), n=24, seed=0):
        self.H, self.G, self.hd = shape
        self.rows, self.n, self.page = rows, n, page
        self.lay = pages_util.Layout(page, self.hd)
        self.ops = PagedKv(*shape, page, pages, width, max_requests=rows, max_tokens=rows * n, rope_half=True)
        self.pool = torch.zeros(pages, self.G, self.lay.part, dtype=torch.uint8, device="cuda")
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
        self.lens, self.refs = dev([0] * rows), dev([0] * pages)
        self.new, self.pos, self.source, self.keep = dev([0] * rows), torch.zeros(rows, n, dtype=torch.int32, device="cuda"), dev(list(range(rows))), dev([1 << 30] * rows)
        g = gen(seed)
        self.qkv = normal(g, rows, n, self.H + 2 * self.G, self.hd)
        self.q, self.out = torch.zeros(rows, n, self.H, self.hd, device="cuda"), torch.zeros(rows, n, self.H, self.hd, device="cuda")

    def step(self):
        p = ptr
        view = self.ops.view(p(self.pool), p(self.table), p(self.lens), self.rows, new_lens=p(self.new))
        self.ops.update(view, p(self.refs), p(self.refs), p(self.table), p(self.lens), source=p(self.source), keep=p(self.keep), add=p(self.new), stream=stream())
        self.ops.append(view, p(self.qkv), self.n, p(self.pos), p(self.q), stream=stream())
        self.ops.attend(view, p(self.q), self.n, p(self.out), stream=stream())

    def set(self, new, source=None, keep=None):
        self.new.copy_(dev(new))
        self.source.copy_(dev(source or list(range(self.rows))))
        self.keep.copy_(dev(keep or [1 << 30] * self.rows))

    def dense(self):
        cap = self.table.shape[1] * self.page
        k = np.zeros((self.rows, self.G, cap, self.hd))
        v = np.zeros_like(k)
        pool, table = self.pool.cpu().numpy(), self.table.tolist()
        for b, n in enumerate(self.lens.tolist()):
            for i in range(-(-n // self.page)):
                k[b, :, i * self.page : (i + 1) * self.page], v[b, :, i * self.page : (i + 1) * self.page] = self.lay.read(pool[table[b][i]])
        return torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()

    def check(self):
        torch.cuda.synchronize()
        new = self.new.tolist()
        ref, tol = kv_util.attend(self.q, *self.dense(), self.lens.tolist(), new)[:2]
        live = torch.arange(self.n, device="cuda")[None] < self.new[:, None]
        assert bool(((self.out.double() - ref).abs() <= tol)[live].all())
        assert self.ops.errors(stream()) == 0


SCRIPT = [([20, 0, 0, 0], None, None), ([1, 1, 1, 1], [0, 0, 0, 0], None), ([1, 1, 1, 1], None, None), ([3, 0, 1, 24], None, [1 << 30, 0, 10, 1 << 30]),
          ([1, 1, 1, 1], [3, 3, 2, 0], None), ([1, 5, 1, 1], None, None)]


def test_sessions_step_by_step():
    s = Sessions()
    for new, source, keep in SCRIPT:
        s.set(new, source, keep)
        s.step()
        s.check()
    # what a row holds does not depend on where: compacted, the next step gives the same bits
    before = s.out.clone()
    used = dev([0])
    s.set([0] * 4, None, [n - m for n, m in zip(s.lens.tolist(), s.new.tolist())])
    s.step()
    s.ops.compact(s.ops.view(ptr(s.pool), ptr(s.table), ptr(s.lens), 4), ptr(s.refs), ptr(s.refs), ptr(s.table), ptr(used), stream=stream())
    s.set(SCRIPT[-1][0])
    s.step()
    s.check()
    live = torch.arange(s.n, device="cuda")[None] < s.new[:, None]
    assert torch.equal(s.out[live], before[live])


def test_sessions_in_a_graph():
    """One captured step follows lengths, rows and tables; eager work in between; every replay against an eager twin."""
    a, b = Sessions(seed=1), Sessions(seed=1)
    side = torch.cuda.Stream()
    a.set([0] * 4)
    with torch.cuda.stream(side):
        a.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        a.step()
    for new, source, keep in SCRIPT:
        for s in (a, b):
            s.set(new, source, keep)
        torch.cuda.synchronize()
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        live = torch.arange(a.n, device="cuda")[None] < a.new[:, None]
        for x in ("pool", "table", "lens", "refs"):
            assert torch.equal(getattr(a, x), getattr(b, x)), x
        assert torch.equal(a.out[live], b.out[live])
        a.check()


def other_arrays(p):
    """The pool's arrays at addresses of 16 bytes and no more, as parts of larger ones."""
    def moved(x, to):
        y = torch.zeros(x.numel() * x.element_size() + 4096, dtype=torch.uint8, device="cuda")[to : to + x.numel() * x.element_size()]
        y = y.view(x.dtype).view(x.shape)
        assert y.data_ptr() % 256 == to % 256
        return y.copy_(x)

    p.pool, p.q, p.out = moved(p.pool, 16), moved(p.q, 48), moved(p.out, 80)
    p.table, p.lens, p.new = moved(p.table, 4), moved(p.lens, 12), moved(p.new, 20)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("hd", [64, 128])
def test_attend_addresses(hd, n, page):
    p = Pool((8, 2, hd), page, [333, 40 + n], [n, n], shared=1, seed=40, width=None if n == 1 else 4000 // page)
    other_arrays(p)
    p.check_all()


def test_graphs_on_one_handle_from_its_first_calls():
    """Attention of one token, of a turn and of a prompt, captured by a handle that has run nothing, two graphs of one
    workspace; replayed in turn, with eager calls, new lengths, tables and queries in between."""
    for n, width in ((1, 40000 // 64), (40, 20000 // 64)):
        p = Pool((32, 8, 128), 64, [5000, 300, 64 + n], [n, n, n], shared=1, seed=50 + n, width=width)
        side = torch.cuda.Stream()
        outs = [torch.full_like(p.out, 7.0) for _ in range(2)]
        queries = [p.q.clone(), p.q.flip(0).contiguous()]
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        torch.cuda.synchronize()
        for graph, q, out in zip(graphs, queries, outs):
            with torch.cuda.graph(graph, stream=side):
                p.ops.attend(p.view(), ptr(q), n, ptr(out), stream=torch.cuda.current_stream().cuda_stream)
        for turn in range(4):
            p.lens_h = [5000 - 700 * turn, 300 - turn, 64 + n]
            p.new_h = [n, n if turn % 2 else 0, n]
            p.lens.copy_(dev(p.lens_h))
            p.new.copy_(dev(p.new_h))
            p.table_h[0][1], p.table_h[0][2] = p.table_h[0][2], p.table_h[0][1]
            p.table.copy_(dev(p.table_h))
            for graph, q, out in zip(graphs, queries, outs):
                q.add_(0.01 * turn)
                out.fill_(7.0)
                graph.replay()
                p.q = q
                p.out = torch.full_like(out, 7.0)
                want = p.expect()
                p.check(p.attend(), want)
                p.check(out, want)
                assert torch.equal(out, p.out)
        assert p.ops.errors(stream()) == 0


def test_rows_in_a_graph_apart():
    """Update and compact of arrays apart (one launch each), captured as a handle's first calls; replayed there and back."""
    rows, page, pages, width = 5, 16, 40, 6
    ops = PagedKv(4, 1, 64, page, pages, width, max_requests=rows, max_tokens=64)
    lay = [dict(table=torch.full((rows, width), -1, dtype=torch.int32, device="cuda"), lens=dev([0] * rows), refs=dev([0] * pages)) for _ in range(3)]
    pool = torch.arange(pages * ops.page_bytes // 4, dtype=torch.int32, device="cuda").view(pages, -1)
    source, keep, add, used = dev(list(range(rows))), dev([1 << 30] * rows), dev([0] * rows), dev([0])
    host = pool.cpu().numpy().copy()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    a, b, c = lay
    with torch.cuda.graph(graph, stream=side):
        at = torch.cuda.current_stream().cuda_stream
        ops.update(ops.view(ptr(pool), ptr(a["table"]), ptr(a["lens"]), rows), ptr(a["refs"]), ptr(b["refs"]), ptr(b["table"]), ptr(b["lens"]),
                   source=ptr(source), keep=ptr(keep), add=ptr(add), stream=at)
        ops.compact(ops.view(ptr(pool), ptr(b["table"]), ptr(b["lens"]), rows), ptr(b["refs"]), ptr(c["refs"]), ptr(c["table"]), ptr(used), stream=at)
    table, lens, refs = [[-1] * width for _ in range(rows)], [0] * rows, [0] * pages
    g = random.Random(3)
    for turn in range(8):
        src = [g.randrange(rows) for _ in range(rows)]
        kp = [g.randint(0, 60) for _ in range(rows)]
        ad = [g.randint(0, 30) for _ in range(rows)]
        source.copy_(dev(src)), keep.copy_(dev(kp)), add.copy_(dev(ad))
        c["table"].fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        table, lens, refs, copies = pages_util.update(table, lens, refs, src, kp, ad, page, width)
        old = host.copy()
        for to, at in copies.items():
            host[to] = old[at]
        table, refs, to, n = pages_util.compact(table, lens, refs, page)
        old = host.copy()
        for x, y in to.items():
            host[y] = old[x]
        assert b["lens"].tolist() == lens and c["refs"].tolist() == refs and int(used) == n
        for row, got, length in zip(table, c["table"].tolist(), lens):
            assert got[: -(-length // page)] == row[: -(-length // page)]
        assert np.array_equal(pool.cpu().numpy(), host)
        a["table"].copy_(c["table"]), a["lens"].copy_(b["lens"]), a["refs"].copy_(c["refs"])
        assert ops.errors(stream()) == 0


def test_two_handles_side_by_side():
    pools = [Pool((32, 8, 128), 64, [3000 + 7 * i, 900], [1, 1], seed=20 + i) for i in range(2)]
    want = [p.attend().clone() for p in pools]
    streams = [torch.cuda.Stream() for _ in pools]
    torch.cuda.synchronize()
    for _ in range(10):
        for p, s in zip(pools, streams):
            p.ops.attend(p.view(), ptr(p.q), p.n, ptr(p.out), stream=s.cuda_stream)
    torch.cuda.synchronize()
    for p, w in zip(pools, want):
        assert torch.equal(p.out, w)


def test_same_bits_every_time():
    p = Pool((32, 8, 128), 64, [5000, 700, 64], [1, 1, 1], seed=30)
    want = p.attend().clone()
    for _ in range(5):
        assert torch.equal(p.attend(), want)


def test_against_dense_f16_caches():
    """The elements are f16 numbers: an f16 cache that holds them gives the same attention."""
    p = Pool((32, 8, 128), 64, [700, 65, 128], [1, 1, 1], seed=31)
    k, v = (x.half() for x in p.dense())
    ops = KvOps(32, 8, 128, max_requests=3, max_tokens=3, kv_f16=True)
    out = torch.full_like(p.out, 7.0)
    ops.attend(ops.view(ptr(k), ptr(v), ptr(p.lens), 3, k.shape[2], new_lens=ptr(p.new)), ptr(p.q), 1, ptr(out), stream=stream())
    torch.cuda.synchronize()
    p.check(out)
    p.check(p.attend())


# --------------------------------------------------------------------------
# refusals
# --------------------------------------------------------------------------
def test_calls_refused():
    p = Pool((8, 2, 64), 16, [9, 9], [2, 2], seed=5)
    x = torch.zeros(1 << 16, device="cuda")
    i32 = torch.zeros(1 << 12, dtype=torch.int32, device="cuda")
    a, q, out = ptr(p.pool), ptr(p.q), ptr(p.out)
    good = (a, ptr(p.table), ptr(p.lens), 2)

    def view(**kw):
        args = dict(zip(("pool", "table", "lens", "requests"), good), **kw)
        return p.ops.view(**args)

    def refused(text, f, *args, **kw):
        with pytest.raises(S2HipError, match=text):
            f(*args, stream=stream(), **kw)

    for bad, text in ((dict(requests=0), "requests"), (dict(requests=3), "requests"), (dict(pool=0), "pool is NULL"), (dict(pool=a + 8), "pool is not aligned"),
                      (dict(table=0), "table"), (dict(lens=0), "lens"), (dict(new_lens=ptr(p.new) + 2), "new_lens")):
        refused(text, p.ops.attend, view(**bad), q, 2, out)
        refused(text, p.ops.append, view(**bad), ptr(x), 2, ptr(i32), out)
    for bad, text in ((dict(n_tokens=0), "n_tokens"), (dict(n_tokens=3), "n_tokens"), (dict(q=0), "q is NULL"), (dict(q=q + 4), "q is not aligned"), (dict(out=0), "out is NULL"),
                      (dict(out=q + 16), "overlaps")):
        refused(text, p.ops.attend, view(), **dict(dict(q=q, n_tokens=2, out=out), **bad))
    rows = 2 * 2 * 64 * 4
    for bad, text in ((dict(n_tokens=3), "n_tokens"), (dict(qkv=0), "qkv"), (dict(positions=0), "positions"), (dict(q_out=0), "q_out"), (dict(q_norm=ptr(x)), "go together"),
                      (dict(q_out=ptr(x) + 16), "q_out overlaps qkv"), (dict(k_held=out + 8 * rows - 16), "k_held overlaps q_out"), (dict(v_held=ptr(x)), "v_held overlaps qkv"),
                      (dict(k_held=ptr(x) + (1 << 17), v_held=ptr(x) + (1 << 17) + 16), "v_held overlaps k_held"), (dict(k_held=ptr(x) + 4), "k_held is not aligned")):
        refused(text, p.ops.append, view(), **dict(dict(qkv=ptr(x), n_tokens=2, positions=ptr(i32), q_out=out), **bad))
    refs, refs_out, table_out, lens_out = (ptr(i32) + 4096 * k for k in range(4))
    base = dict(refs=refs, refs_out=refs_out, table_out=table_out, lens_out=lens_out)
    for bad, text in ((dict(refs=0), "refs"), (dict(refs_out=0), "refs_out"), (dict(table_out=0), "table_out"), (dict(lens_out=0), "lens_out"), (dict(refs_out=refs + 4), "refs_out overlaps"),
                      (dict(table_out=ptr(p.table) + 4), "table_out overlaps"), (dict(lens_out=ptr(p.lens) + 4), "lens_out overlaps"), (dict(layers=0), "layers"),
                      (dict(layers=1025), "layers"), (dict(layers=2, layer_stride=64), "layer_stride"), (dict(layers=2, layer_stride=p.pages * p.ops.page_bytes + 8), "layer_stride"),
                      (dict(source=2), "source"), (dict(keep=ptr(i32) + 1), "keep"), (dict(add=3), "add"), (dict(refs_out=table_out), "overlap"), (dict(lens_out=refs), "overlap"),
                      (dict(table_out=refs_out + 16), "overlap"), (dict(add=refs_out), "overlap"), (dict(source=table_out, keep=ptr(i32)), "overlap")):
        refused(text, p.ops.update, view(), **dict(base, **bad))
    base = dict(refs=refs, refs_out=refs_out, table_out=table_out, used_out=lens_out)
    for bad, text in ((dict(refs=0), "refs"), (dict(used_out=0), "used_out"), (dict(layers=0), "layers"), (dict(moved_to=2), "moved_to"), (dict(used_out=refs_out), "overlap"),
                      (dict(moved_to=table_out), "overlap"), (dict(used_out=ptr(p.lens)), "overlap")):
        refused(text, p.ops.compact, view(), **dict(base, **bad))
    torch.cuda.synchronize()
    assert p.ops.errors(stream()) == 0
    p.check(p.attend())


def test_overlaps_refused():
    """Every output against every array of its call, by its last and its first word; and apart by none it goes."""
    H, G, hd, page, pages, width, R, n = 4, 2, 64, 16, 6, 3, 2, 2
    ops = PagedKv(H, G, hd, page, pages, width, max_requests=R, max_tokens=R * n)
    rows, pool = R * n, pages * ops.page_bytes
    base = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    spare = [ptr(base) + 65536 * (i + 4) for i in range(12)]  # the pool lies in front of them

    up = lambda x: -(-x // 16) * 16  # noqa: E731

    def check(call, sizes, outputs, same=()):
        """call(addresses): arrays of `sizes` bytes by name; those of `outputs` share nothing with the others but for the pairs `same`."""
        where = dict(zip(sizes, spare), pool=ptr(base))
        call(where)
        for out in outputs:
            for other in sizes:
                if out == other or (other, out) in same:
                    continue
                for at in (where[other] + up(1 - sizes[out]), where[other] + (sizes[other] - 4) // 16 * 16):
                    if at >= ptr(base):
                        with pytest.raises(S2HipError, match="overlap"):
                            call(dict(where, **{out: at}))
                for at in (where[other] - up(sizes[out]), where[other] + up(sizes[other])):
                    if at >= ptr(base) and out != "pool":
                        call(dict(where, **{out: at}))

    def view(w):
        return ops.view(w["pool"], w["table"], w["lens"], R, new_lens=w.get("new_lens", 0))

    q, kv = rows * H * hd * 4, rows * G * hd * 4
    batch = dict(table=R * width * 4, lens=4 * R, new_lens=4 * R, pool=pool)
    check(lambda w: ops.append(view(w), w["qkv"], n, w["positions"], w["q_out"], q_norm=w["q_norm"], k_norm=w["k_norm"], k_held=w["k_held"], v_held=w["v_held"], stream=stream()),
          dict(batch, qkv=q + 2 * kv, positions=rows * 4, q_norm=hd * 4, k_norm=hd * 4, q_out=q, k_held=kv, v_held=kv), ["q_out", "k_held", "v_held", "pool"])
    check(lambda w: ops.attend(view(w), w["q"], n, w["out"], stream=stream()), dict(batch, q=q, out=q), ["out"])
    batch = dict(table=R * width * 4, lens=4 * R, pool=pool, refs=4 * pages, refs_out=4 * pages, table_out=R * width * 4)
    check(lambda w: ops.update(view(w), w["refs"], w["refs_out"], w["table_out"], w["lens_out"], source=w["source"], keep=w["keep"], add=w["add"], stream=stream()),
          dict(batch, lens_out=4 * R, source=4 * R, keep=4 * R, add=4 * R), ["refs_out", "table_out", "lens_out", "pool"], [("lens", "lens_out")])
    check(lambda w: ops.compact(view(w), w["refs"], w["refs_out"], w["table_out"], w["used_out"], moved_to=w["moved_to"], stream=stream()),
          dict(batch, used_out=4, moved_to=4 * pages), ["refs_out", "table_out", "used_out", "moved_to", "pool"])
    # layers apart: what lies between them is the caller's, what lies in one is not
    where = dict(zip(("table", "lens", "refs"), spare), pool=ptr(base))
    gap = up(pool)

    def grow(refs_out):
        ops.update(ops.view(where["pool"], where["table"], where["lens"], R), where["refs"], refs_out, spare[8], spare[9], layers=3, layer_stride=gap + 1024, stream=stream())

    for at in (gap, gap + 1024 - 4 * pages, 2 * gap + 1024, 3 * gap + 2048):
        grow(ptr(base) + at)
    for at in (0, gap - 4, gap + 1024 - 4, gap + 1024, 2 * gap + 1020, 2 * gap + 2048 - 4 * pages + 4, 3 * gap + 2044):
        with pytest.raises(S2HipError, match="refs_out overlaps pool"):
            grow(ptr(base) + at)
    torch.cuda.synchronize()
    ops.errors(stream())


def test_errors_refused_under_capture():
    p = Pool((8, 2, 64), 16, [9], [1], seed=5)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        p.ops.attend(p.view(), ptr(p.q), 1, ptr(p.out), stream=torch.cuda.current_stream().cuda_stream)
        with pytest.raises(S2HipError, match="captured"):
            p.ops.errors(torch.cuda.current_stream().cuda_stream)
    graph.replay()
    torch.cuda.synchronize()
    p.check(p.out)
