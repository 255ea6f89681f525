"""KV-cache operators (s2hip.KvOps) against 64-bit computations: sizes around
the tiles' borders, ragged and idle requests, strided caches, values that must
not be seen, ties, graphs and streams."""

import math

import numpy as np
import pytest
import torch

import kv_util
from s2hip import KvOps, S2HipError
from s2hip.kvops import ERR_F16_RANGE, ERR_LENS, ERR_POSITION

pytestmark = pytest.mark.gpu
U = kv_util.U


@pytest.fixture(autouse=True)
def float32_tensors():
    """Whatever another module has made the default type."""
    was = torch.get_default_dtype()
    torch.set_default_dtype(torch.float32)
    yield
    torch.set_default_dtype(was)


SHAPES = {"gqa4": (32, 8, 128), "tiny": (8, 2, 64), "mha": (4, 4, 64), "gqa3": (6, 2, 128), "gqa7": (14, 2, 128)}


def dev(x, dtype=None):
    return torch.as_tensor(x, dtype=dtype).cuda()


def normal(g, *shape, spread=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * spread


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def stream():
    return torch.cuda.current_stream().cuda_stream


def ptr(x):
    return 0 if x is None else x.data_ptr()


class Batch:
    """Random caches of a batch with lens / new given, and the call's arrays."""

    def __init__(self, shape, f16, lens, new, cap=None, prefix=0, seed=0, spread=1.5, rows=None):
        self.H, self.G, self.hd = shape
        self.f16, self.R, self.n = f16, len(lens), rows or max(1, max(new))
        self.cap = cap or max(1, max(lens))
        self.P = prefix
        g = gen(seed)
        dt = torch.float16 if f16 else torch.float32
        self.k = normal(g, self.R, self.G, self.cap, self.hd).to(dt)
        self.v = normal(g, self.R, self.G, self.cap, self.hd).to(dt)
        self.pk = normal(g, self.G, prefix, self.hd).to(dt) if prefix else None
        self.pv = normal(g, self.G, prefix, self.hd).to(dt) if prefix else None
        self.q = normal(g, self.R, self.n, self.H, self.hd, spread=spread)
        self.out = torch.full_like(self.q, 7.0)
        self.lens_h, self.new_h = list(lens), list(new)
        self.lens, self.new = dev(lens, torch.int32), dev(new, torch.int32)
        self.ops = KvOps(self.H, self.G, self.hd, max_requests=max(self.R, 1), max_tokens=max(self.R * self.n, 1), kv_f16=f16)

    def view(self, **kw):
        return self.ops.view(ptr(self.k), ptr(self.v), ptr(self.lens), self.R, self.cap, new_lens=ptr(self.new), prefix_k=ptr(self.pk),
                             prefix_v=ptr(self.pv), prefix_len=self.P, **kw)

    def attend(self):
        self.ops.attend(self.view(), ptr(self.q), self.n, ptr(self.out), stream=stream())
        torch.cuda.synchronize()
        return self.out

    def expect(self):
        return kv_util.attend(self.q, self.k, self.v, self.lens_h, self.new_h, self.pk, self.pv)

    def check(self, out, want=None):
        ref, tol = (want or self.expect())[:2]
        live = torch.arange(self.n, device="cuda")[None] < self.new[:, None]
        assert bool((out[~live] == 7.0).all()), "rows of no token were written"
        far = (out.double() - ref).abs()[live]
        assert bool((far <= tol[live]).all()), f"off by {far.max().item():.3g}, {(far / tol[live]).max().item():.3g} of the bound"

    def check_all(self):
        self.check(self.attend())
        assert self.ops.errors(stream()) == 0


# --------------------------------------------------------------------------
# attend
# --------------------------------------------------------------------------
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_attend_step(shape, f16):
    lens = [1, 2, 15, 16, 17, 33, 100]
    Batch(SHAPES[shape], f16, lens, [1] * 7, cap=128, prefix=45, seed=1).check_all()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000])
def test_attend_lengths(length, f16):
    """One request's own cache alone, and the same length as the prefix."""
    Batch((8, 2, 64), f16, [length], [1], seed=length).check_all()
    Batch((8, 2, 128), f16, [1, 3], [1, 1], prefix=length, seed=length).check_all()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("requests", [1, 2, 4, 5, 8, 9, 16])
def test_attend_requests(requests, f16):
    lens = [1 + (37 * b) % 90 for b in range(requests)]
    Batch((32, 8, 128), f16, lens, [1] * requests, cap=96, prefix=333, seed=requests).check_all()


# Capacities: of the size of the lengths, and so large that a call counts as much work (it is launched by capacities)
ROOM = [None, 32768]


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("n", [2, 3, 4, 5, 7, 8, 9, 16, 31, 32, 33, 64, 65, 130])
def test_attend_several_tokens(n, f16, room):
    """Causal within the new tokens; ragged; an idle request between others."""
    new = [n, max(1, n // 2), 0, 1, n]
    lens = [n, n // 2 + 40, 9, 1, n + 77]
    Batch((8, 2, 128), f16, lens, new, cap=room or n + 80, prefix=70, seed=n).check_all()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("n,prefix", [(8, 1000), (9, 2500), (33, 0), (40, 64), (200, 63), (380, 65), (500, 1)])
def test_attend_splits(n, prefix, f16):
    """From many splits of a row tile to one, tiles that end inside a split."""
    Batch((32, 8, 128), f16, [n + 3, n], [n, n - 5], cap=9000, prefix=prefix, seed=n).check_all()


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("case", ["prompt", "turns", "turns64", "mha", "gqa7"])
def test_attend_many_tokens(case, f16, room):
    shape, lens, new, P = {
        "prompt": ((8, 2, 128), [517], [517], 0),
        "turns": ((32, 8, 128), [250, 300, 131, 250], [250, 221, 130, 3], 700),
        "turns64": ((8, 2, 64), [250, 300, 131], [250, 221, 130], 257),
        "mha": ((4, 4, 64), [300, 129], [300, 128], 33),
        "gqa7": ((14, 2, 128), [200, 77], [190, 77], 100),
    }[case]
    Batch(shape, f16, lens, new, cap=room or max(lens) + 5, prefix=P, seed=5).check_all()


@pytest.mark.parametrize("f16", [False, True])
def test_attend_long(f16):
    """Few rows over long caches: the work is split over the keys."""
    Batch((8, 2, 128), f16, [20011, 3], [1, 1], cap=20100, prefix=9001, seed=3).check_all()


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("n", [1, 40])
def test_attend_sharp_scores(n, f16, room):
    """Large scores: one key takes nearly everything."""
    Batch((8, 2, 128), f16, [n + 60, n + 5], [n, n], cap=room, prefix=150, seed=8, spread=12.0).check_all()


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("n", [1, 70])
def test_attend_wide_range_f32(n, room):
    """f32 values far outside the f16 range, keys small to match; rows of very different size."""
    b = Batch((8, 2, 128), False, [n + 60, n + 5], [n, n], cap=room, prefix=150, seed=9)
    for x in (b.k, b.pk):
        x.mul_(1e-6)
    b.q.mul_(1e6)
    for x in (b.v, b.pv):
        x.mul_(1e7)
    b.v[0, :, 3] *= 1e-9
    b.check_all()


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("n", [1, 70])
def test_attend_zero_rows(n, f16, room):
    """Queries, keys or values of zeros: equal weights, outputs of zero."""
    b = Batch((8, 2, 64), f16, [n + 60, n + 5], [n, n], cap=room, prefix=40, seed=9)
    b.q[0] = 0
    b.k[1] = 0
    b.v[1] = 0
    b.pv[0] = 0
    b.check_all()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("n", [1, 3, 40, 150])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("room", ROOM)
def test_attend_does_not_see(room, bad, n, f16):
    """Slots not in use, an idle request's cache and later tokens' keys and
    values hold NaN or infinities: rows that do not see them are as without."""
    b = Batch((8, 2, 128), f16, [n + 21, n, 30, n + 40], [n, n, 0, n], cap=room or n + 64, prefix=50, seed=n)
    want = b.expect()
    for r, used in enumerate(b.lens_h):
        b.k[r, :, used:] = bad
        b.v[r, :, used:] = bad
    b.k[2], b.v[2] = bad, bad
    b.check(b.attend(), want)
    # the last token of request 0 brings a value that is no number: its own row alone holds one, in that dim alone
    b.v[0, :, n + 20, 3] = bad
    out = b.attend().clone()
    assert not bool(out[0, n - 1, :, 3].isfinite().any())
    out[0, n - 1, :, 3] = want[0][0, n - 1, :, 3].float()
    b.check(out, want)
    # and a key: its whole row holds none
    b.k[0, :, n + 20] = math.nan
    out = b.attend().clone()
    assert bool(out[0, n - 1].isnan().all())
    out[0, n - 1] = want[0][0, n - 1].float()
    b.check(out, want)
    # a value of the prefix: that dim of every row
    b.k[0, :, n + 20], b.v[0, :, n + 20, 3] = 0.5, 0.5
    b.pv[1, 49, 7] = bad
    out = b.attend()
    live = torch.arange(n, device="cuda")[None] < b.new[:, None]
    half = b.H // b.G
    assert not bool(out[live][:, half:, 7].isfinite().any()) and bool(out[live][:, :half].isfinite().all())
    assert bool(out[live][:, half:, :7].isfinite().all()) and bool(out[live][:, half:, 8:].isfinite().all())


@pytest.mark.parametrize("f16", [False, True])
def test_attend_strided(f16):
    """Token-major caches ([slot][kv head][dim]) inside larger arrays, a prefix with spare room."""
    b = Batch((8, 2, 128), f16, [70, 33], [5, 1], cap=80, prefix=60, seed=4)
    g = b.G
    big_k = torch.full((2, 80, g + 1, 128 + 16), math.nan, dtype=b.k.dtype, device="cuda")
    big_v = big_k.clone()
    big_k[:, :, :g, :128] = b.k.permute(0, 2, 1, 3)
    big_v[:, :, :g, :128] = b.v.permute(0, 2, 1, 3)
    room_k = torch.full((g, 77, 128), math.nan, dtype=b.k.dtype, device="cuda")
    room_v = room_k.clone()
    room_k[:, :60], room_v[:, :60] = b.pk, b.pv
    s = big_k.stride()
    view = b.ops.view(ptr(big_k), ptr(big_v), ptr(b.lens), 2, 80, new_lens=ptr(b.new), prefix_k=ptr(room_k), prefix_v=ptr(room_v),
                      prefix_len=60, prefix_capacity=77, request_stride=s[0], head_stride=s[2], slot_stride=s[1])
    b.ops.attend(view, ptr(b.q), b.n, ptr(b.out), stream=stream())
    torch.cuda.synchronize()
    b.check(b.out)


def test_attend_default_new_lens():
    """new_lens NULL: every request brings n_tokens, one of length 0 none."""
    b = Batch((8, 2, 64), False, [4, 0, 9], [3, 0, 3], cap=12, seed=2)
    view = b.ops.view(ptr(b.k), ptr(b.v), ptr(b.lens), 3, 12)
    b.ops.attend(view, ptr(b.q), 3, ptr(b.out), stream=stream())
    torch.cuda.synchronize()
    b.check(b.out)
    assert b.ops.errors(stream()) == 0


def test_attend_requests_out_of_range():
    """Values that do not fit leave their request out and are reported; the others are served."""
    lens, new = [5, 13, -1, 6, 6], [1, 1, 1, 7, 2]
    b = Batch((8, 2, 64), True, [5, 0, 0, 0, 6], [1, 0, 0, 0, 2], cap=12, seed=2, rows=3)
    b.lens.copy_(dev(lens, torch.int32))
    bad_new = dev(new, torch.int32)
    b.ops.attend(b.ops.view(ptr(b.k), ptr(b.v), ptr(b.lens), 5, 12, new_lens=ptr(bad_new)), ptr(b.q), 3, ptr(b.out), stream=stream())
    torch.cuda.synchronize()
    b.check(b.out)
    assert b.ops.errors(stream()) == ERR_LENS
    assert b.ops.errors(stream()) == 0


def test_attend_far_offsets():
    """A request whose cache lies past 2^31 elements, and past 2^32 bytes."""
    R, G, cap, hd = 66, 8, 32768, 128
    n = R * G * cap * hd
    k = torch.empty(n, dtype=torch.float16, device="cuda")
    v = torch.empty(n, dtype=torch.float16, device="cuda")
    b = Batch((8, 8, 128), True, [32768], [1], cap=cap, seed=6)
    kk, vv = kv_util.dense(k, R, G, cap, hd), kv_util.dense(v, R, G, cap, hd)
    kk[65], vv[65] = b.k[0], b.v[0]
    lens = torch.zeros(R, dtype=torch.int32, device="cuda")
    lens[65] = 32768
    q = torch.zeros(R, 1, 8, hd, device="cuda")
    q[65] = b.q[0]
    out = torch.full_like(q, 7.0)
    ops = KvOps(8, 8, hd, max_requests=R, max_tokens=R, kv_f16=True)
    ops.attend(ops.view(ptr(k), ptr(v), ptr(lens), R, cap), ptr(q), 1, ptr(out), stream=stream())
    torch.cuda.synchronize()
    assert bool((out[:65] == 7.0).all())
    b.check(out[65:])


@pytest.mark.parametrize("f16", [False, True])
def test_attend_same_bits(f16):
    b = Batch((32, 8, 128), f16, [500, 77, 300], [1, 1, 1], prefix=800, seed=11)
    first = b.attend().clone()
    for _ in range(5):
        assert torch.equal(b.attend(), first)


# --------------------------------------------------------------------------
# attend_weigh
# --------------------------------------------------------------------------
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("case", ["step", "step_prefix", "step16", "step64", "few", "turns", "prompt", "mha", "long"])
def test_weigh(case, f16, room):
    shape, lens, new, P = {
        "step": ((32, 8, 128), [1, 2, 70, 129, 300], [1] * 5, 0),
        "step_prefix": ((8, 2, 64), [1, 40, 0, 17], [1, 1, 0, 1], 77),
        "step64": ((32, 8, 128), [3 + 5 * b for b in range(64)], [1] * 64, 33),
        "step16": ((32, 8, 128), [3 + 5 * b for b in range(16)], [1] * 16, 257),
        "few": ((6, 2, 128), [40, 3, 65], [3, 2, 1], 31),
        "turns": ((8, 2, 128), [150, 90, 33], [130, 77, 33], 100),
        "prompt": ((32, 8, 128), [333], [333], 0),
        "mha": ((4, 4, 64), [70, 150], [64, 150], 129),
        "long": ((8, 2, 128), [9001, 40], [1, 1], 2003),
    }[case]
    if room and len(lens) > 16:
        room = 600  # (as much work, less memory)
    b = Batch(shape, f16, lens, new, cap=room or max(lens) + 9, prefix=P, seed=12)
    want = b.expect()
    g = gen(3)
    w_in, pw_in = normal(g, b.R, b.G, b.cap).abs(), normal(g, b.G, max(P, 1)).abs()
    w = torch.full_like(w_in, 5.0)
    pw = torch.full_like(pw_in, 5.0)

    def go(w_in, w, pw_in, pw):
        b.out.fill_(7.0)
        b.ops.attend_weigh(b.view(), ptr(b.q), b.n, ptr(b.out), ptr(w), weights_in=ptr(w_in), prefix_weights_out=ptr(pw),
                           prefix_weights_in=ptr(pw_in), stream=stream())
        torch.cuda.synchronize()

    def hold(w, base, tol, ref, used):
        far = (w.double() - base - ref).abs()
        assert bool((far <= tol + U * (base + ref))[used].all())

    used = torch.arange(b.cap, device="cuda")[None, None] < b.lens[:, None, None]
    used = used.expand(w.shape)
    go(w_in, w, pw_in if P else None, pw if P else None)
    b.check(b.out, want)
    assert bool((w[~used] == 5.0).all())
    hold(w, w_in.double(), want[3], want[2], used)
    if P:
        hold(pw, pw_in.double(), want[5], want[4], torch.ones_like(pw, dtype=torch.bool))
    # the same bits again, in place, and from nothing; the prefix left out
    w2, pw2 = w_in.clone(), pw_in.clone()
    go(w2, w2, pw2 if P else None, pw2 if P else None)
    assert torch.equal(w2[used], w[used]) and torch.equal(w2[~used], w_in[~used])
    assert not P or torch.equal(pw2, pw)
    go(None, w, None, None)
    hold(w, torch.zeros_like(w).double(), want[3], want[2], used)
    # every row gives away a weight of one
    rows = sum(b.new_h) * b.H // b.G
    given = w.double().masked_fill(~used, 0).sum((0, 2)) + want[4].sum(1)
    assert bool(((given - rows).abs() <= 1e-4 * rows).all())
    assert b.ops.errors(stream()) == 0


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("n", [1, 3, 50])
def test_weigh_does_not_see(n, f16, room):
    b = Batch((8, 2, 128), f16, [n + 21, n, 30, n + 40], [n, n, 0, n], cap=room or n + 64, prefix=50, seed=n)
    want = b.expect()
    for r, used in enumerate(b.lens_h):
        b.k[r, :, used:] = math.nan
        b.v[r, :, used:] = math.nan
    b.k[2], b.v[2] = math.nan, math.nan
    w = torch.zeros(b.R, b.G, b.cap, device="cuda")
    pw = torch.zeros(b.G, b.P, device="cuda")
    b.ops.attend_weigh(b.view(), ptr(b.q), b.n, ptr(b.out), ptr(w), prefix_weights_out=ptr(pw), stream=stream())
    torch.cuda.synchronize()
    b.check(b.out, want)
    assert bool(((w.double() - want[2]).abs() <= want[3]).all()) and bool(((pw.double() - want[4]).abs() <= want[5]).all())
    # a key that is no number takes with it the weights of the keys that its token sees, and of no others
    b.k[0, :, n + 20] = math.nan
    b.ops.attend_weigh(b.view(), ptr(b.q), b.n, ptr(b.out), ptr(w), prefix_weights_out=ptr(pw), stream=stream())
    torch.cuda.synchronize()
    assert bool(w[0, :, : n + 21].isnan().all()) and bool(pw.isnan().all())
    assert bool(((w.double() - want[2]).abs() <= want[3])[1:].all())
    b.k[0, :, n + 20], b.k[1, :, n - 1] = 0.25, math.nan
    b.new[1] = 0  # the request sits out: no row sees that key
    b.ops.attend_weigh(b.view(), ptr(b.q), b.n, ptr(b.out), ptr(w), prefix_weights_out=ptr(pw), stream=stream())
    torch.cuda.synchronize()
    assert bool(pw.isfinite().all()) and bool((w[1, :, :n] == 0).all())


# --------------------------------------------------------------------------
# append
# --------------------------------------------------------------------------
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_append(shape, norm, f16):
    H, G, hd = SHAPES[shape]
    n, new, lens, cap = 6, [6, 1, 0, 3], [6, 20, 5, 23], 23
    g = gen(1)
    dt = torch.float16 if f16 else torch.float32
    qkv = normal(g, 4, n, H + 2 * G, hd, spread=3.0)
    positions = torch.randint(0, 32768, (4, n), generator=g, device="cuda", dtype=torch.int32)
    positions[0, 0], positions[0, 1], positions[3, 2] = 0, 32767, 2**31 - 1
    gq, gk = (normal(g, hd, spread=0.3) + 1, normal(g, hd, spread=0.3) + 1) if norm else (None, None)
    k, v = normal(g, 4, G, cap, hd).to(dt), normal(g, 4, G, cap, hd).to(dt)
    q = torch.full((4, n, H, hd), 7.0, device="cuda")
    scores = torch.full((4, G, cap), 5.0, device="cuda")
    where = torch.full((4, G, cap), -5, dtype=torch.int32, device="cuda")
    k0, v0 = k.clone(), v.clone()
    lens_d, new_d = dev(lens, torch.int32), dev(new, torch.int32)
    ops = KvOps(H, G, hd, max_requests=4, max_tokens=4 * n, kv_f16=f16, rope_base=1e6, eps=1e-6)
    ops.append(ops.view(ptr(k), ptr(v), ptr(lens_d), 4, cap, new_lens=ptr(new_d)), ptr(qkv), n, ptr(positions), ptr(q), q_norm=ptr(gq),
               k_norm=ptr(gk), scores=ptr(scores), slot_positions=ptr(where), stream=stream())
    torch.cuda.synchronize()
    wq = kv_util.rotated(qkv[:, :, :H], positions, gq, 1e6, 1e-6)
    wk = kv_util.rotated(qkv[:, :, H : H + G], positions, gk, 1e6, 1e-6)
    # norm: the mean of hd squares and its root within (log2(hd) + 6) U, two products; rotation: cos and sin within
    # 2 U and the angle's 64-bit rounding (2 pi 2^-53 of the turns: 2.2e-7 at 2^31 / 2 pi of them), two products, a sum
    size = lambda x: x.abs().view(*x.shape[:-1], hd // 2, 2).sum(-1).repeat_interleave(2, -1)  # noqa: E731
    rel = 24 * U + 2 * math.pi * 2.0**-52 * positions.double()[..., None, None]
    for b in range(4):
        t, lo = new[b], lens[b] - new[b]
        assert bool((q[b, t:] == 7.0).all())
        assert bool(((q[b, :t].double() - wq[b, :t]).abs() <= 1.5 * size(wq[b, :t]) * rel[b, :t]).all())
        touched = torch.zeros(cap, dtype=torch.bool, device="cuda")
        touched[lo : lo + t] = True
        assert torch.equal(k[b, :, ~touched], k0[b, :, ~touched]) and torch.equal(v[b, :, ~touched], v0[b, :, ~touched])
        assert bool((scores[b, :, ~touched] == 5).all()) and bool((where[b, :, ~touched] == -5).all())
        if t:
            gk_ = k[b, :, lo : lo + t].transpose(0, 1).double()
            half = 2.0**-11 if f16 else 0.0  # f16: half a step more
            far = (gk_ - wk[b, :t]).abs()
            assert bool((far <= 1.5 * size(wk[b, :t]) * rel[b, :t] + half * wk[b, :t].abs() + (2.0**-25 if f16 else 0)).all())
            assert torch.equal(v[b, :, lo : lo + t].transpose(0, 1), qkv[b, :t, H + G :].to(dt))
            assert bool((scores[b, :, lo : lo + t] == 0).all())
            assert torch.equal(where[b, :, lo : lo + t], positions[b, :t].expand(G, t))
    assert ops.errors(stream()) == 0


def test_append_reports():
    """A negative position leaves its token out; a length that does not fit its request; f16 overflow is told."""
    H, G, hd, cap = 4, 2, 64, 8
    qkv = normal(gen(2), 3, 2, H + 2 * G, hd)
    qkv[0, 0, H + G, 5] = 7e4
    positions = dev([[3, -1], [0, 1], [5, 6]], torch.int32)
    lens = dev([2, 9, 2], torch.int32)
    k = torch.full((3, G, cap, hd), 9.0, dtype=torch.float16, device="cuda")
    v = k.clone()
    q = torch.full((3, 2, H, hd), 7.0, device="cuda")
    ops = KvOps(H, G, hd, max_requests=3, max_tokens=6, kv_f16=True)
    ops.append(ops.view(ptr(k), ptr(v), ptr(lens), 3, cap), ptr(qkv), 2, ptr(positions), ptr(q), stream=stream())
    torch.cuda.synchronize()
    assert ops.errors(stream()) == ERR_LENS | ERR_POSITION | ERR_F16_RANGE
    assert bool((q[0, 1] == 7).all()) and bool((q[1] == 7).all()) and not bool((q[2] == 7).any())
    assert bool((k[0, :, 1:] == 9).all()) and bool((k[1] == 9).all()) and bool((v[1] == 9).all())
    assert v[0, 0, 0, 5].item() == math.inf and torch.equal(v[2, :, :2].transpose(0, 1), qkv[2, :, H + G :].half())


# --------------------------------------------------------------------------
# evict
# --------------------------------------------------------------------------
def run_evict(ops, k, v, lens, keep, recent, sinks, scores, positions, layers=1, in_place=False):
    LR, G, cap, _ = k.shape
    R = LR // layers
    lens_d = dev(lens, torch.int32)
    if in_place:
        so, po, lo = scores, positions, lens_d
    else:
        so, po, lo = torch.full_like(scores, -3.0), torch.full_like(positions, -3), torch.full_like(lens_d, -3)
    before = [x.clone() for x in (k, v, scores, positions, so, po)]
    ops.evict(ops.view(ptr(k), ptr(v), ptr(lens_d), R, cap), keep, recent, sinks, ptr(scores), ptr(positions), ptr(so), ptr(po), ptr(lo),
              layers=layers, stream=stream())
    torch.cuda.synchronize()
    k0, v0, s0, p0, wso, wpo = before
    sn, pn = s0.cpu().numpy(), p0.cpu().numpy()
    for i in range(LR):
        for g in range(G):
            come, to, m = kv_util.select(sn[i, g], pn[i, g], lens[i % R], keep, recent, sinks)
            wso[i, g, :m], wpo[i, g, :m] = s0[i, g, :m], p0[i, g, :m]
            for x, y in ((k0, k0), (v0, v0), (wso, s0), (wpo, p0)):
                x[i, g, to] = y[i, g, come]
    bits = lambda x: x.contiguous().view(torch.int16 if x.element_size() == 2 else torch.int32)  # noqa: E731
    for got, want in ((k, k0), (v, v0), (so, wso), (po, wpo)):
        assert torch.equal(bits(got), bits(want))
    assert lo.tolist() == [min(n, keep) for n in lens]
    return lo


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("cap,keep,recent,sinks", [(1, 1, 0, 0), (2, 1, 1, 0), (40, 7, 3, 2), (64, 64, 5, 0), (1000, 999, 0, 4), (1024, 1, 0, 1),
                                                   (1025, 300, 100, 4), (4096, 1024, 1020, 4), (4097, 2048, 0, 0), (17000, 5000, 128, 4), (32768, 16384, 1, 4)])
def test_evict_sizes(cap, keep, recent, sinks, in_place):
    g = gen(cap + keep)
    lens = [cap, max(1, cap - 1), min(cap, keep + 1), min(cap, keep), 0]
    k, v = normal(g, 5, 2, cap, 64), normal(g, 5, 2, cap, 64)
    scores = normal(g, 5, 2, cap, spread=2.0).exp()
    positions = torch.argsort(torch.rand(5, 2, cap, generator=g, device="cuda"), 2).to(torch.int32) + 3
    ops = KvOps(2, 2, 64, max_requests=5, max_tokens=5)
    run_evict(ops, k, v, lens, keep, recent, sinks, scores, positions, in_place=in_place)
    assert ops.errors(stream()) == 0


@pytest.mark.parametrize("values", ["equal", "coarse", "zeros", "special", "negative"])
def test_evict_ties_and_odd_scores(values):
    g = gen(7)
    cap = 700
    x = normal(g, 3, 2, cap)
    scores = {
        "equal": torch.ones_like(x),
        "coarse": (x * 2).round(),
        "zeros": torch.where(x > 0, torch.zeros_like(x), -torch.zeros_like(x)),
        "special": torch.where(x > 1, math.nan, torch.where(x > 0.5, math.inf, torch.where(x < -1, -math.inf, x))),
        "negative": -x.exp(),
    }[values].contiguous()
    positions = torch.arange(cap, dtype=torch.int32, device="cuda").expand(3, 2, cap).contiguous()
    k, v = normal(g, 3, 2, cap, 128).half(), normal(g, 3, 2, cap, 128).half()
    ops = KvOps(2, 2, 128, max_requests=3, max_tokens=3, kv_f16=True)
    run_evict(ops, k, v, [700, 650, 211], 210, 31, 4, scores, positions)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("layers,cap", [(1, 900), (9, 300), (40, 130), (40, 2100)])
def test_evict_many_caches(layers, cap, in_place):
    """From few caches to more than two a compute unit."""
    g = gen(layers)
    R, G = 4, 4
    scores = normal(g, layers * R, G, cap).abs()
    positions = torch.argsort(torch.rand(layers * R, G, cap, generator=g, device="cuda"), 2).to(torch.int32)
    k, v = normal(g, layers * R, G, cap, 128).half(), normal(g, layers * R, G, cap, 128).half()
    ops = KvOps(4, 4, 128, max_requests=R, max_tokens=R, kv_f16=True)
    run_evict(ops, k, v, [cap, cap // 2, cap // 3, 0], cap // 2 - 5, 20, 4, scores, positions, layers=layers, in_place=in_place)


def test_evict_positions_given_twice():
    """More safe slots than room: the heaviest of them stay."""
    g = gen(9)
    scores = normal(g, 1, 2, 90)
    positions = torch.full((1, 2, 90), 5, dtype=torch.int32, device="cuda")
    positions[0, 1, 60:] = -(2**31)
    k, v = normal(g, 1, 2, 90, 64), normal(g, 1, 2, 90, 64)
    run_evict(KvOps(2, 2, 64, max_requests=1, max_tokens=1), k, v, [90], 40, 3, 0, scores, positions)


def test_evict_layers_strided():
    """Layers in one call equal one call per layer; rows with gaps between them."""
    g = gen(10)
    LR, G, cap = 6, 2, 300
    scores = normal(g, LR, G, cap).abs()
    positions = torch.arange(cap, dtype=torch.int32, device="cuda").expand(LR, G, cap).contiguous()
    k, v = normal(g, LR, G, cap, 64).half(), normal(g, LR, G, cap, 64).half()
    ops = KvOps(2, 2, 64, max_requests=2, max_tokens=2, kv_f16=True)
    k2, v2, s2, p2 = k.clone(), v.clone(), scores.clone(), positions.clone()
    run_evict(ops, k, v, [300, 201], 111, 20, 4, scores, positions, layers=3)
    big_k = torch.zeros(LR, cap, G, 80, dtype=torch.float16, device="cuda")
    big_v = big_k.clone()
    big_k[..., :64], big_v[..., :64] = k2.permute(0, 2, 1, 3), v2.permute(0, 2, 1, 3)
    st = big_k.stride()
    lens = dev([300, 201], torch.int32)
    for layer in range(3):
        at = slice(2 * layer, 2 * layer + 2)
        lo = torch.zeros(2, dtype=torch.int32, device="cuda")
        view = ops.view(ptr(big_k[at]), ptr(big_v[at]), ptr(lens), 2, cap, request_stride=st[0], head_stride=st[2], slot_stride=st[1])
        ops.evict(view, 111, 20, 4, ptr(s2[at]), ptr(p2[at]), ptr(s2[at]), ptr(p2[at]), ptr(lo), stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(big_k[..., :64].permute(0, 2, 1, 3), k) and torch.equal(big_v[..., :64].permute(0, 2, 1, 3), v)
    assert bool((big_k[..., 64:] == 0).all()) and lo.tolist() == [111, 111]


def test_evict_out_of_range():
    g = gen(11)
    k, v = normal(g, 2, 2, 50, 64), normal(g, 2, 2, 50, 64)
    scores, positions = normal(g, 2, 2, 50), torch.arange(50, dtype=torch.int32, device="cuda").expand(2, 2, 50).contiguous()
    lens, lo = dev([51, 40], torch.int32), dev([-3, -3], torch.int32)
    before = [x[0].clone() for x in (k, v, scores, positions)]
    ops = KvOps(2, 2, 64, max_requests=2, max_tokens=2)
    ops.evict(ops.view(ptr(k), ptr(v), ptr(lens), 2, 50), 10, 2, 1, ptr(scores), ptr(positions), ptr(scores), ptr(positions), ptr(lo), stream=stream())
    torch.cuda.synchronize()
    assert lo.tolist() == [-3, 10] and ops.errors(stream()) == ERR_LENS
    assert all(torch.equal(x[0], y) for x, y in zip((k, v, scores, positions), before))


# --------------------------------------------------------------------------
# together
# --------------------------------------------------------------------------
class Serve:
    """Requests over one shared prefix: append, attend with weights, evict."""

    def __init__(self, f16, R=3, cap=64, P=70, seed=0, shape=(8, 2, 64)):
        self.H, self.G, self.hd = shape
        self.R, self.cap, self.P = R, cap, P
        g = self.g = gen(seed)
        dt = torch.float16 if f16 else torch.float32
        self.k = torch.full((R, self.G, cap, self.hd), math.nan, dtype=dt, device="cuda")
        self.v = self.k.clone()
        self.pk, self.pv = normal(g, self.G, P, self.hd).to(dt), normal(g, self.G, P, self.hd).to(dt)
        self.scores = torch.full((R, self.G, cap), math.nan, device="cuda")
        self.where = torch.full((R, self.G, cap), -9, dtype=torch.int32, device="cuda")
        self.gq, self.gk = normal(g, self.hd, spread=0.2) + 1.5, normal(g, self.hd, spread=0.2) + 1
        self.lens = torch.zeros(R, dtype=torch.int32, device="cuda")
        self.new = torch.zeros(R, dtype=torch.int32, device="cuda")
        self.ops = KvOps(self.H, self.G, self.hd, max_requests=R, max_tokens=R * cap, kv_f16=f16)
        self.view = self.ops.view(ptr(self.k), ptr(self.v), ptr(self.lens), R, cap, new_lens=ptr(self.new), prefix_k=ptr(self.pk),
                                  prefix_v=ptr(self.pv), prefix_len=P)

    def buffers(self, n):
        return (torch.zeros(self.R, n, self.H + 2 * self.G, self.hd, device="cuda"), torch.zeros(self.R, n, dtype=torch.int32, device="cuda"),
                torch.zeros(self.R, n, self.H, self.hd, device="cuda"), torch.zeros(self.R, n, self.H, self.hd, device="cuda"))

    def step(self, qkv, positions, q, out):
        n, s = qkv.shape[1], stream()
        self.ops.append(self.view, ptr(qkv), n, ptr(positions), ptr(q), q_norm=ptr(self.gq), k_norm=ptr(self.gk), scores=ptr(self.scores),
                        slot_positions=ptr(self.where), stream=s)
        self.ops.attend_weigh(self.view, ptr(q), n, ptr(out), ptr(self.scores), weights_in=ptr(self.scores), stream=s)

    def cut(self, keep, recent, sinks):
        self.ops.evict(self.view, keep, recent, sinks, ptr(self.scores), ptr(self.where), ptr(self.scores), ptr(self.where), ptr(self.lens),
                       stream=stream())


@pytest.mark.parametrize("f16", [False, True])
def test_serve_turns_and_cuts(f16):
    """Turns, decode steps and cuts; every attention against 64 bits on the caches as they then are, every
    cut against the selection by the scores as they then are."""
    s = Serve(f16)
    nexts = [s.P] * s.R
    for turn, (n, new) in enumerate([(20, [20, 11, 0]), (1, [1, 1, 1]), (30, [30, 30, 5]), (1, [1, 1, 1]), (1, [1, 0, 1]), (25, [3, 25, 25]), (1, [1, 1, 1])]):
        qkv, positions, q, out = s.buffers(n)
        qkv.copy_(normal(s.g, *qkv.shape))
        positions.copy_(dev([[p + t for t in range(n)] for p in nexts], torch.int32))
        nexts = [p + t for p, t in zip(nexts, new)]
        old = s.scores.clone()
        s.new.copy_(dev(new, torch.int32))
        s.lens.add_(s.new)
        out.fill_(7.0)
        s.step(qkv, positions, q, out)
        torch.cuda.synchronize()
        lens = s.lens.tolist()
        ref, tol, w, wt, _, _ = kv_util.attend(q, s.k, s.v, lens, new, s.pk, s.pv)
        for b in range(s.R):
            assert bool(((out[b, : new[b]].double() - ref[b, : new[b]]).abs() <= tol[b, : new[b]]).all())
            assert bool((out[b, new[b] :] == 7).all())
            base = old[b, :, : lens[b]].double()
            base[:, lens[b] - new[b] :] = 0
            got = s.scores[b, :, : lens[b]].double()
            assert bool(((got - base - w[b, :, : lens[b]]).abs() <= wt[b, :, : lens[b]] + U * got).all())
        if max(lens) > 32:
            k, v, sc, wh = (x.clone() for x in (s.k, s.v, s.scores, s.where))
            s.cut(24, 8, s.P + 2)  # the first two own positions count as sinks
            torch.cuda.synchronize()
            assert s.lens.tolist() == [min(24, x) for x in lens]
            for b in range(s.R):
                for g in range(s.G):
                    come, to, m = kv_util.select(sc[b, g].cpu().numpy(), wh[b, g].cpu().numpy(), lens[b], 24, 8, s.P + 2)
                    for x in (k, v, sc, wh):
                        x[b, g, to] = x[b, g, come].clone()
                    assert torch.equal(s.where[b, g, :m], wh[b, g, :m]) and torch.equal(s.scores[b, g, :m], sc[b, g, :m])
                    assert torch.equal(s.k[b, g, :m], k[b, g, :m]) and torch.equal(s.v[b, g, :m], v[b, g, :m])
    assert s.ops.errors(stream()) == 0


@pytest.mark.parametrize("f16", [False, True])
def test_prefix_filled_by_the_operators(f16):
    """A prompt prefilled as one request, used as the prefix of two: as if each had its own copy."""
    H, G, hd, P, n = 8, 2, 128, 150, 9
    g = gen(21)
    dt = torch.float16 if f16 else torch.float32
    ops = KvOps(H, G, hd, max_requests=2, max_tokens=512, kv_f16=f16)
    pk, pv = torch.zeros(G, 200, hd, dtype=dt, device="cuda"), torch.zeros(G, 200, hd, dtype=dt, device="cuda")
    one = dev([P], torch.int32)
    qkv, pos = normal(g, 1, P, H + 2 * G, hd), torch.arange(P, dtype=torch.int32, device="cuda")[None].contiguous()
    q0 = torch.zeros(1, P, H, hd, device="cuda")
    ops.append(ops.view(ptr(pk), ptr(pv), ptr(one), 1, 200), ptr(qkv), P, ptr(pos), ptr(q0), stream=stream())
    qkv2 = normal(g, 2, n, H + 2 * G, hd)
    pos2 = (P + torch.arange(n, dtype=torch.int32, device="cuda")).expand(2, n).contiguous()
    lens, k, v, q = dev([n, n], torch.int32), torch.zeros(2, G, 20, hd, dtype=dt, device="cuda"), torch.zeros(2, G, 20, hd, dtype=dt, device="cuda"), torch.zeros(2, n, H, hd, device="cuda")
    view = ops.view(ptr(k), ptr(v), ptr(lens), 2, 20, prefix_k=ptr(pk), prefix_v=ptr(pv), prefix_len=P, prefix_capacity=200)
    ops.append(view, ptr(qkv2), n, ptr(pos2), ptr(q), stream=stream())
    out = torch.zeros_like(q)
    ops.attend(view, ptr(q), n, ptr(out), stream=stream())
    whole_k, whole_v = torch.zeros(2, G, 180, hd, dtype=dt, device="cuda"), torch.zeros(2, G, 180, hd, dtype=dt, device="cuda")
    for a, b, c in ((whole_k, pk, k), (whole_v, pv, v)):
        a[:, :, :P], a[:, :, P : P + n] = b[:, :P], c[:, :, :n]
    full, new = dev([P + n] * 2, torch.int32), dev([n, n], torch.int32)
    copy = torch.zeros_like(q)
    ops.attend(ops.view(ptr(whole_k), ptr(whole_v), ptr(full), 2, 180, new_lens=ptr(new)), ptr(q), n, ptr(copy), stream=stream())
    torch.cuda.synchronize()
    ref, tol = kv_util.attend(q, k, v, [n, n], [n, n], pk[:, :P], pv[:, :P])[:2]
    assert bool(((out.double() - ref).abs() <= tol).all()) and bool(((copy.double() - ref).abs() <= tol).all())


def test_graph_replays_follow_lens():
    """One captured step replayed as the requests grow, with eager work between, against an eager twin."""
    a, b = Serve(True, seed=5), Serve(True, seed=5)
    bufs = a.buffers(1)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        a.new.fill_(0)
        a.step(*bufs)  # nothing to do: loads the code
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        a.step(*bufs)
    for i in range(30):
        qkv = normal(a.g, *bufs[0].shape)
        normal(b.g, *bufs[0].shape)
        live = [1, int(i % 3 != 0), int(i > 4)]
        for x, held in ((a, bufs), (b, b.buffers(1))):
            held[0].copy_(qkv)
            held[1].copy_((x.lens + x.P)[:, None])
            x.new.copy_(dev(live, torch.int32))
            x.lens.add_(x.new)
            if x is a:
                graph.replay()
            else:
                x.step(*held)
                torch.cuda.synchronize()
                got = held[3]
        torch.cuda.synchronize()
        for r in range(3):
            if live[r]:
                assert torch.equal(bufs[3][r], got[r])
                assert torch.equal(a.scores[r, :, : int(a.lens[r])], b.scores[r, :, : int(b.lens[r])])
        if i == 20:
            for x in (a, b):
                x.cut(10, 4, 0)
    assert a.ops.errors(stream()) == 0


def test_graph_of_a_cut():
    a = Serve(False, seed=6)
    g = gen(4)
    a.k.copy_(normal(g, *a.k.shape))
    a.v.copy_(normal(g, *a.v.shape))
    a.where.copy_(torch.arange(a.cap, dtype=torch.int32, device="cuda"))
    so, po, lo = torch.zeros_like(a.scores), torch.zeros_like(a.where), torch.zeros_like(a.lens)

    def cut():
        a.ops.evict(a.view, 20, 5, 2, ptr(a.scores), ptr(a.where), ptr(so), ptr(po), ptr(lo), stream=stream())

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        cut()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        cut()
    for i in range(4):
        a.scores.copy_(normal(g, *a.scores.shape))
        a.lens.copy_(dev([60, 64, 20 + i], torch.int32))
        k, sc, wh = a.k.clone(), a.scores.clone(), a.where.clone()
        graph.replay()
        torch.cuda.synchronize()
        lens = a.lens.tolist()
        assert lo.tolist() == [min(x, 20) for x in lens]
        for b in range(a.R):
            for j in range(a.G):
                come, to, m = kv_util.select(sc[b, j].cpu().numpy(), wh[b, j].cpu().numpy(), lens[b], 20, 5, 2)
                k[b, j, to] = k[b, j, come].clone()
                sc[b, j, to] = sc[b, j, come].clone()
                assert torch.equal(so[b, j, :m], sc[b, j, :m])
        assert torch.equal(a.k, k)


def test_two_handles_on_two_streams():
    """Handles of their own run side by side."""
    x, y = Batch((32, 8, 128), True, [900, 3], [1, 1], prefix=1500, seed=1), Batch((32, 8, 128), True, [40, 700], [33, 33], prefix=900, seed=2)
    want = x.expect(), y.expect()
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        for b, s in zip((x, y), streams):
            with torch.cuda.stream(s):
                b.ops.attend(b.view(), ptr(b.q), b.n, ptr(b.out), stream=s.cuda_stream)
    torch.cuda.synchronize()
    x.check(x.out, want[0])
    y.check(y.out, want[1])


# --------------------------------------------------------------------------
# refusals
# --------------------------------------------------------------------------
def refused(match, call, *args, **kw):
    with pytest.raises(S2HipError, match=match):
        call(*args, **kw)


def test_refusals():
    b = Batch((8, 2, 64), True, [4, 4], [2, 2], cap=8, prefix=5, seed=1)
    o, v = b.ops, b.view
    p = {n: ptr(getattr(b, n)) for n in ("k", "v", "q", "out", "lens", "new", "pk", "pv")}
    for heads, kv, hd, kw, match in [
        (8, 3, 64, {}, "multiple of kv_heads"), (8, 0, 64, {}, "multiple of kv_heads"), (130, 2, 64, {}, "not supported"),
        (8, 2, 96, {}, "head_dim 96"), (8, 2, 64, {"max_requests": 0}, "max_requests"), (8, 2, 64, {"max_requests": 257}, "max_requests"),
        (8, 2, 64, {"max_tokens": 0}, "max_tokens"), (8, 2, 64, {"rope_base": 0.0}, "rope_base"), (8, 2, 64, {"rope_base": math.nan}, "rope_base"),
        (8, 2, 64, {"eps": -1.0}, "eps"), (8, 2, 64, {"scale": math.inf}, "scale"), (8, 2, 64, {"device": 99}, "device 99")]:
        refused(match, KvOps, heads, kv, hd, **kw)
    refused("requests 3", o.attend, o.view(p["k"], p["v"], p["lens"], 3, 8), p["q"], 1, p["out"])
    refused("requests 0", o.attend, o.view(p["k"], p["v"], p["lens"], 0, 8), p["q"], 1, p["out"])
    refused("max_tokens 4", o.attend, v(), p["q"], 3, p["out"])
    refused("n_tokens 0", o.attend, v(), p["q"], 0, p["out"])
    refused("capacity 0", o.attend, o.view(p["k"], p["v"], p["lens"], 2, 0), p["q"], 1, p["out"])
    refused("capacity 32769", o.attend, o.view(p["k"], p["v"], p["lens"], 2, 32769), p["q"], 1, p["out"])
    refused("k is NULL", o.attend, o.view(0, p["v"], p["lens"], 2, 8), p["q"], 1, p["out"])
    refused("v is not aligned", o.attend, o.view(p["k"], p["v"] + 2, p["lens"], 2, 8), p["q"], 1, p["out"])
    refused("lens is NULL", o.attend, o.view(p["k"], p["v"], 0, 2, 8), p["q"], 1, p["out"])
    refused("prefix_k is NULL", o.attend, o.view(p["k"], p["v"], p["lens"], 2, 8, prefix_len=5), p["q"], 1, p["out"])
    refused("prefix_len 32769", o.attend, o.view(p["k"], p["v"], p["lens"], 2, 8, prefix_k=p["pk"], prefix_v=p["pv"], prefix_len=32769), p["q"], 1, p["out"])
    refused("prefix_capacity 4", o.attend, v(prefix_capacity=4), p["q"], 1, p["out"])
    refused("slot_stride 4 is not a multiple", o.attend, v(slot_stride=4), p["q"], 1, p["out"])
    refused("slot_stride 56 is below", o.attend, v(slot_stride=56), p["q"], 1, p["out"])
    refused("prefix_slot_stride 8 is below", o.attend, v(prefix_slot_stride=8), p["q"], 1, p["out"])
    refused("q is NULL", o.attend, v(), 0, 1, p["out"])
    refused("out is not aligned", o.attend, v(), p["q"], 1, p["out"] + 4)
    refused("out overlaps q", o.attend, v(), p["q"], 2, p["q"])
    refused("NULL argument", o.attend, None, p["q"], 1, p["out"])
    refused("weights_out is NULL", o.attend_weigh, v(), p["q"], 1, p["out"], 0)
    refused("prefix_weights_in without", o.attend_weigh, v(), p["q"], 1, p["out"], p["k"], prefix_weights_in=p["k"])
    refused("qkv is NULL", o.append, v(), 0, 1, p["lens"], p["q"])
    refused("positions is NULL", o.append, v(), p["q"], 1, 0, p["q"])
    refused("q_norm and k_norm", o.append, v(), p["q"], 1, p["lens"], p["out"], q_norm=p["q"])
    refused("keep is 0", o.evict, v(), 0, 0, 0, *([p["q"]] * 5))
    refused("recent 6 is more than keep 5", o.evict, v(), 5, 6, 0, *([p["q"]] * 5))
    refused("layers 0", o.evict, v(), 5, 3, 2, *([p["q"]] * 5), layers=0)
    refused("layer_stride 3", o.evict, v(), 5, 3, 2, *([p["q"]] * 5), layers=2, layer_stride=3)
    refused("scores_out overlaps", o.evict, v(), 5, 3, 2, p["q"], p["k"], p["q"] + 4, p["k"], p["out"])
    refused("positions_out overlaps", o.evict, v(), 5, 3, 2, p["q"], p["k"], p["q"], p["k"] + 4, p["out"])
    refused("lens_out overlaps", o.evict, v(), 5, 3, 2, *([p["q"]] * 4), p["lens"] + 4)
    refused("weights_out overlaps", o.attend_weigh, v(), p["q"], 1, p["out"], p["k"], weights_in=p["k"] + 4)
    refused("lens_out is NULL", o.evict, v(), 5, 3, 2, *([p["q"]] * 4), 0)
    torch.cuda.synchronize()
    b.check(b.attend())  # nothing was launched, the handle works


def test_refusals_of_layouts():
    """Strides that make rows overlap, or that are too large; arrays that overlap."""
    b = Batch((8, 2, 64), True, [4, 4], [2, 2], cap=8, prefix=5, seed=1)
    o, v = b.ops, b.view
    p = {n: ptr(getattr(b, n)) for n in ("k", "v", "q", "out", "lens")}
    call = (p["q"], 1, p["out"])
    refused("slot_stride 16777216 is not below", o.attend, v(slot_stride=1 << 24), *call)
    refused("prefix_slot_stride 16777216 is not below", o.attend, v(prefix_slot_stride=1 << 24), *call)
    refused("request_stride 1099511627776 is too large", o.attend, v(request_stride=1 << 40), *call)
    refused("overlap", o.attend, v(request_stride=1016), *call)
    refused("overlap", o.attend, v(head_stride=504), *call)
    refused("overlap", o.attend, v(slot_stride=128, head_stride=120), *call)
    refused("overlap", o.append, v(slot_stride=128, head_stride=64, request_stride=128), p["k"], 1, p["lens"], p["q"])
    five = (p["q"], p["k"], p["q"], p["k"], p["out"])
    refused("overlap", o.evict, v(), 5, 3, 2, *five, layers=2, layer_stride=2040)
    refused("overlap", o.evict, v(slot_stride=256, head_stride=64, request_stride=128), 5, 3, 2, *five, layers=2, layer_stride=256)
    refused("q_out overlaps qkv", o.append, v(), p["q"], 1, p["lens"], p["q"])
    refused("q_out overlaps qkv", o.append, v(), p["q"], 1, p["lens"], p["q"] + 4 * 2 * 12 * 64 - 16)
    torch.cuda.synchronize()
    b.check(b.attend())


@pytest.mark.parametrize("f16", [False, True])
def test_strides_left_out(f16):
    """Slots before heads: the strides left out step over what the given ones lay out."""
    b = Batch((8, 2, 64), f16, [30, 41, 9], [2, 3, 1], cap=48, seed=12)
    dense = b.attend().clone()
    k, v = b.k.transpose(1, 2).contiguous(), b.v.transpose(1, 2).contiguous()
    out = torch.full_like(b.q, 7.0)
    view = b.ops.view(ptr(k), ptr(v), ptr(b.lens), 3, 48, new_lens=ptr(b.new), head_stride=64, slot_stride=128)
    b.ops.attend(view, ptr(b.q), b.n, ptr(out), stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(out, dense)


def test_evict_layer_stride_left_out():
    """Layers of [slot][request][kv head] rows, and more requests than tokens of a call."""
    g = gen(13)
    L, R, G, cap = 3, 2, 2, 100
    scores = normal(g, L * R, G, cap).abs()
    positions = torch.arange(cap, dtype=torch.int32, device="cuda").expand(L * R, G, cap).contiguous()
    k, v = normal(g, L * R, G, cap, 64), normal(g, L * R, G, cap, 64)
    ops = KvOps(2, 2, 64, max_requests=2, max_tokens=1)
    k2, v2 = (x.reshape(L, R, G, cap, 64).permute(0, 3, 1, 2, 4).contiguous() for x in (k, v))
    s2, p2, lens, lo = scores.clone(), positions.clone(), dev([100, 61], torch.int32), dev([0, 0], torch.int32)
    run_evict(ops, k, v, [100, 61], 40, 8, 2, scores, positions, layers=L)
    view = ops.view(ptr(k2), ptr(v2), ptr(lens), R, cap, request_stride=128, head_stride=64, slot_stride=256)
    ops.evict(view, 40, 8, 2, ptr(s2), ptr(p2), ptr(s2), ptr(p2), ptr(lo), layers=L, stream=stream())
    torch.cuda.synchronize()
    for x, y in ((k, k2), (v, v2)):
        assert torch.equal(x.reshape(L, R, G, cap, 64).permute(0, 3, 1, 2, 4), y)
    assert lo.tolist() == [40, 40]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("requests,n,heads,kv,prefix,length", [
    (4, 4, 4, 4, 700, 140), (17, 1, 2, 2, 130, 300), (31, 1, 2, 2, 129, 5), (8, 1, 8, 2, 127, 1), (8, 4, 4, 4, 128, 257), (33, 1, 3, 3, 300, 70),
    (4, 16, 4, 4, 100, 129), (5, 13, 2, 2, 90, 260), (2, 32, 4, 4, 0, 128), (1, 33, 4, 4, 65, 40), (16, 4, 32, 8, 2000, 33), (51, 5, 2, 2, 40, 6),
    (257 // 2, 2, 4, 2, 50, 3), (171, 3, 2, 2, 30, 3)])
def test_weigh_rows(requests, n, heads, kv, prefix, length, f16):
    """Numbers of rows around those where a key's rows are summed by more lanes, or the scores are computed once more; some idle."""
    lens = [max(1, length - b % 5) for b in range(requests)]
    new = [min(lens[b], n - b % n) if b % 4 != 3 else 0 for b in range(requests)]
    b = Batch((heads, kv, 64), f16, lens, new, prefix=prefix, seed=requests + n, rows=n, cap=max(lens) + 3)
    ref = b.expect()
    w, pw = torch.full((b.R, b.G, b.cap), 5.0, device="cuda"), torch.full((b.G, max(prefix, 1)), 5.0, device="cuda")
    b.ops.attend_weigh(b.view(), ptr(b.q), b.n, ptr(b.out), ptr(w), prefix_weights_out=ptr(pw) if prefix else 0, stream=stream())
    torch.cuda.synchronize()
    b.check(b.out, ref)
    used = (torch.arange(b.cap, device="cuda")[None, None] < b.lens[:, None, None]).expand(w.shape)
    assert bool((w[~used] == 5.0).all())
    assert bool(((w.double() - ref[2]).abs() <= ref[3] + U * ref[2])[used].all())
    assert not prefix or bool(((pw.double() - ref[4]).abs() <= ref[5] + U * ref[4]).all())
    assert b.ops.errors(stream()) == 0


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("shape", ["gqa4", "mha", "gqa7"])
@pytest.mark.parametrize("n", [40, 255, 256, 257, 513, 1100])
def test_weigh_chunks(n, shape, f16):
    """Turns whose rows are summed in chunks, around whole blocks of keys, next to a shorter one."""
    b = Batch(SHAPES[shape], f16, [n, n // 3 + 50], [n, n // 3], cap=n + 70, seed=n)
    ref = b.expect()
    w = torch.full((2, b.G, b.cap), 5.0, device="cuda")
    b.ops.attend_weigh(b.view(), ptr(b.q), b.n, ptr(b.out), ptr(w), stream=stream())
    torch.cuda.synchronize()
    b.check(b.out, ref)
    used = (torch.arange(b.cap, device="cuda")[None, None] < b.lens[:, None, None]).expand(w.shape)
    assert bool((w[~used] == 5.0).all())
    assert bool(((w.double() - ref[2]).abs() <= ref[3] + U * ref[2])[used].all())


@pytest.mark.parametrize("low,high", [(-60, 60), (60, -60), (-100, 20), (0, 120)])
@pytest.mark.parametrize("n", [192, 1])
def test_attend_scales_far_apart(n, low, high):
    """f32 caches: values of the first half of the keys 2^low, of the second 2^high; every output within the bound."""
    b = Batch((32, 8, 128), False, [192], [n], prefix=320, cap=32768, seed=3)
    b.pv.mul_(2.0 ** low)
    b.v.mul_(2.0 ** high)
    out = b.attend()
    ref = b.expect()[0]
    assert bool(out.isfinite().all())
    p = kv_util.attend(b.q, b.k, torch.ones_like(b.v), b.lens_h, b.new_h, b.pk, torch.zeros_like(b.pv))[0]  # each row's weight on the second half
    # 2^-20 of each half's part for products, sums and weights as in the plain bound; 2^-38 of the largest value for what falls below it
    bound = 2.0 ** -20 * 8 * (p * 2.0 ** high + (1 - p) * 2.0 ** low) + 2.0 ** -38 * 8 * 2.0 ** max(low, high)
    assert bool(((out.double() - ref).abs() <= bound).all())


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("requests,n,heads,kv,prefix", [(8, 64, 8, 2, 20), (1, 683, 6, 2, 9), (1, 512, 8, 2, 0), (1, 513, 8, 2, 0), (9, 57, 8, 2, 33), (2, 1024, 2, 2, 5)])
def test_weigh_rows_of_turns(requests, n, heads, kv, prefix, f16):
    """Rows up to those whose scores are kept, and a few more."""
    lens = [n + 3 * b for b in range(requests)]
    new = [n - 7 * b for b in range(requests)]
    b = Batch((heads, kv, 64), f16, lens, new, prefix=prefix, seed=n, rows=n)
    ref = b.expect()
    w, pw = torch.full((b.R, b.G, b.cap), 5.0, device="cuda"), torch.full((b.G, max(prefix, 1)), 5.0, device="cuda")
    b.ops.attend_weigh(b.view(), ptr(b.q), b.n, ptr(b.out), ptr(w), prefix_weights_out=ptr(pw) if prefix else 0, stream=stream())
    torch.cuda.synchronize()
    b.check(b.out, ref)
    used = (torch.arange(b.cap, device="cuda")[None, None] < b.lens[:, None, None]).expand(w.shape)
    assert bool((w[~used] == 5.0).all())
    assert bool(((w.double() - ref[2]).abs() <= ref[3] + U * ref[2])[used].all())
    assert not prefix or bool(((pw.double() - ref[4]).abs() <= ref[5] + U * ref[4]).all())


@pytest.mark.parametrize("size", [0.0, 1e-25, 1e25])
def test_append_norm_of_extreme_rows(size):
    """Rows of zeros, and ones whose squares leave f32: as y / sqrt(mean(y^2) + eps) gives them in f32."""
    H, G, hd = 8, 2, 64
    g = gen(21)
    qkv = normal(g, 1, 3, H + 2 * G, hd) * size
    k, v, q = torch.zeros(1, G, 4, hd, device="cuda"), torch.zeros(1, G, 4, hd, device="cuda"), torch.full((1, 3, H, hd), 7.0, device="cuda")
    ones, pos, lens = torch.ones(hd, device="cuda"), torch.zeros(1, 3, dtype=torch.int32, device="cuda"), dev([3], torch.int32)
    ops = KvOps(H, G, hd, max_requests=1, max_tokens=3)
    ops.append(ops.view(ptr(k), ptr(v), ptr(lens), 1, 4), ptr(qkv), 3, ptr(pos), ptr(q), q_norm=ptr(ones), k_norm=ptr(ones), stream=stream())
    torch.cuda.synchronize()
    want = qkv * torch.rsqrt((qkv * qkv).mean(-1, keepdim=True) + 1e-6)
    assert bool(((q - want[:, :, :H]).abs() <= 2.0**-20 * want[:, :, :H].abs()).all())
    assert torch.equal(v[:, :, :3].transpose(1, 2), qkv[:, :, H + G :]) and ops.errors(stream()) == 0


def weigh(b, prefix=True):
    """(weights, prefix weights) of the batch's call, from zero; out in b.out."""
    w, pw = torch.zeros(b.R, b.G, b.cap, device="cuda"), torch.zeros(b.G, max(b.P, 1), device="cuda")
    b.out.fill_(7.0)
    b.ops.attend_weigh(b.view(), ptr(b.q), b.n, ptr(b.out), ptr(w), prefix_weights_out=ptr(pw) if prefix and b.P else 0, stream=stream())
    torch.cuda.synchronize()
    return w, pw


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("size", [2.0**20, 2.0**38, 1e30, 3e38])
@pytest.mark.parametrize("hd,n", [(64, 1), (128, 1), (64, 40), (128, 40), (128, 150)])
def test_attend_does_not_see_large_values(hd, n, size, f16, room):
    """Finite keys and values far above the others in later tokens' slots, in
    slots not in use and in other requests' caches: the rows that do not see
    them keep their bits."""
    size = min(size, 6e4) if f16 else size
    b = Batch((8, 2, hd), f16, [n + 21, n, 30, n + 43], [n, n, 0, n], cap=room or n + 64, prefix=50, seed=n)
    want = b.expect()
    clean = b.attend().clone()
    b.check(clean, want)
    g = gen(99)
    for r, used in enumerate(b.lens_h):
        b.k[r, :, used:] = size
        b.v[r, :, used:] = -size
    b.k[2], b.v[2] = size, size
    # the last tokens of requests 0 and 1 bring large keys and values, seen by their own rows alone
    for r in (0, 1):
        sign = torch.where(torch.rand(b.G, hd, generator=g, device="cuda") < 0.5, -1.0, 1.0)
        b.k[r, :, b.lens_h[r] - 1] = (sign * size).to(b.k.dtype)
        b.v[r, :, b.lens_h[r] - 1] = (-sign * size).to(b.v.dtype)
    b.out.fill_(7.0)
    out = b.attend().clone()
    for r in (0, 1):
        out[r, n - 1] = clean[r, n - 1]
    b.check(out, want)
    assert torch.equal(out, clean)


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("size", [2.0**20, 2.0**38, 1e30])
@pytest.mark.parametrize("hd,n", [(64, 1), (128, 3), (64, 50), (128, 50), (128, 150)])
def test_weigh_does_not_see_large_keys(hd, n, size, f16, room):
    """Large keys in the last tokens' slots, in slots not in use and in an idle
    request's cache: the weights that the tokens before them give are those
    without.  (The last tokens' queries are zeros, so that theirs are known.)"""
    size = min(size, 6e4) if f16 else size
    b = Batch((8, 2, hd), f16, [n + 21, n, 30, n + 43], [n, n, 0, n], cap=room or n + 64, prefix=50, seed=n)
    g = gen(99)
    for r in range(4):
        b.q[r, n - 1] = 0
        b.k[r, :, b.lens_h[r] :] = size
        if r != 3:
            sign = torch.where(torch.rand(b.G, hd, generator=g, device="cuda") < 0.5, -1.0, 1.0)
            b.k[r, :, b.lens_h[r] - 1] = (sign * size).to(b.k.dtype)
    b.k[2] = size
    want = b.expect()
    w, pw = weigh(b)
    b.check(b.out, want)
    used = (torch.arange(b.cap, device="cuda")[None, None] < b.lens[:, None, None]).expand(w.shape)
    assert bool(((w.double() - want[2]).abs() <= want[3] + U * want[2])[used].all())
    assert bool(((pw.double() - want[4]).abs() <= want[5] + U * want[4]).all())


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("n", [1, 3, 50, 130])
def test_weigh_splits_of_no_number(n, f16, room):
    """Keys of no number that fill whole splits of the work: the rows that see
    them give no key a weight that is a number."""
    b = Batch((8, 2, 128), f16, [n + 21, n], [n, n], cap=room or n + 64, prefix=2500, seed=n)
    want = b.expect()
    b.pk[0] = math.nan
    w, pw = weigh(b)
    half = b.H // b.G
    assert bool(b.out[:, :, :half].isnan().all())
    assert bool(w[0, 0, : n + 21].isnan().all()) and bool(w[1, 0, :n].isnan().all()) and bool(pw[0].isnan().all())
    b.out[:, :, :half] = want[0][:, :, :half].float()
    b.check(b.out, want)
    assert bool(((w[:, 1].double() - want[2][:, 1]).abs() <= want[3][:, 1]).all())
    assert bool(((pw[1].double() - want[4][1]).abs() <= want[5][1]).all())


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
@pytest.mark.parametrize("n", [1, 3, 40, 150])
def test_attend_sees_infinite_key(n, bad, f16, room):
    """A key that holds an infinity makes the rows that see it no number, with
    either sign of its score, and the weights of the keys that they see; no others."""
    b = Batch((8, 2, 128), f16, [n + 21, n, 30, n + 40], [n, n, 0, n], cap=room or n + 64, prefix=50, seed=n)
    want = b.expect()
    b.k[0, 1, n + 20, 5] = bad  # request 0's last token alone sees it
    b.k[3, 0, 7, 100] = bad  # all of request 3's rows
    half = b.H // b.G
    for weighed in (False, True):
        b.out.fill_(7.0)
        if weighed:
            w, pw = weigh(b)
        out = b.out.clone() if weighed else b.attend().clone()
        assert bool(out[0, n - 1, half:].isnan().all()) and bool(out[3, :, :half].isnan().all())
        out[0, n - 1, half:], out[3, :, :half] = want[0][0, n - 1, half:].float(), want[0][3, :, :half].float()
        b.check(out, want)
    assert bool(w[0, 1, : n + 21].isnan().all()) and bool(w[3, 0, : n + 40].isnan().all()) and bool(pw.isnan().all())
    for r, j in ((0, 0), (1, 0), (1, 1), (3, 1)):
        assert bool(((w[r, j].double() - want[2][r, j]).abs() <= want[3][r, j]).all())


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("n", [1, 2, 33, 150])
def test_attend_sees_infinite_keys_alone(n, f16, room):
    """Rows all of whose scores are -infinity are no number, and so are the weights; the one-slot row among them."""
    b = Batch((8, 2, 64), f16, [n, n], [n, n], cap=room, seed=n)
    want = b.expect()
    b.q[0].abs_()
    b.k[0] = 0.0
    b.k[0, :, :, 3] = -math.inf
    out = b.attend().clone()
    assert bool(out[0].isnan().all())
    out[0] = want[0][0].float()
    b.check(out, want)
    w, _ = weigh(b)
    assert bool(b.out[0].isnan().all()) and bool(w[0, :, :n].isnan().all())
    assert bool(((w[1].double() - want[2][1]).abs() <= want[3][1]).all())


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("up", [-76, -100, 60, 100])
@pytest.mark.parametrize("n", [1, 50, 150])
def test_attend_small_keys_large_queries(n, up, room):
    """f32 caches: queries times 2^up over keys times 2^-up, and values that small: as without."""
    b = Batch((8, 2, 128), False, [n + 60, n + 5], [n, n], cap=room, prefix=150, seed=9)
    clean = b.expect()
    b.q.mul_(2.0**up)
    b.k.mul_(2.0**-up)
    b.pk.mul_(2.0**-up)
    w, pw = weigh(b)
    b.check(b.out, clean)
    b.check(b.attend(), clean)
    assert bool(((w.double() - clean[2]).abs() <= clean[3] + U * clean[2]).all())
    assert bool(((pw.double() - clean[4]).abs() <= clean[5] + U * clean[4]).all())


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("up", [-74, -60, 100])
@pytest.mark.parametrize("n", [1, 50, 150])
def test_attend_values_of_any_size(n, up, room):
    """f32 caches: values times 2^up give outputs times 2^up."""
    b = Batch((8, 2, 128), False, [n + 60, n + 5], [n, n], cap=room, prefix=150, seed=9)
    want = b.expect()
    b.v.mul_(2.0**up)
    b.pv.mul_(2.0**up)
    out = b.attend()
    live = torch.arange(n, device="cuda")[None] < b.new[:, None]
    b.check(torch.where(live[:, :, None, None], out * 2.0**-up, out), want)


@pytest.mark.parametrize("cap", [130, 32768])
@pytest.mark.parametrize("f16", [False, True])
def test_one_token_of_many_heads(f16, cap):
    """One token of 32 and of 64 heads over one: as many rows as a turn, in caches of the lengths' size and in large ones."""
    for H, lens in (((64, 2, 64), [101, 1, 130]), ((64, 1, 128), [40, 77, 9])):
        b = Batch(H, f16, lens, [1] * 3, cap=cap, prefix=300, seed=31)
        want = b.expect()
        b.check(b.attend(), want)
        w, pw = weigh(b)
        b.check(b.out, want)
        used = (torch.arange(b.cap, device="cuda")[None, None] < b.lens[:, None, None]).expand(w.shape)
        assert bool(((w.double() - want[2]).abs() <= want[3] + U * want[2])[used].all())
        assert bool(((pw.double() - want[4]).abs() <= want[5] + U * want[4]).all())


@pytest.mark.parametrize("f16", [False, True])
def test_step_weights_computed_once_more(f16):
    """A step in caches so large that its scores are not kept."""
    b = Batch((32, 2, 64), f16, [1 + 9 * r for r in range(33)], [1] * 33, cap=32768, prefix=257, seed=32)
    want = b.expect()
    w, pw = weigh(b)
    b.check(b.out, want)
    used = (torch.arange(b.cap, device="cuda")[None, None] < b.lens[:, None, None]).expand(w.shape)
    assert bool(((w.double() - want[2]).abs() <= want[3] + U * want[2])[used].all())
    assert bool(((pw.double() - want[4]).abs() <= want[5] + U * want[4]).all())


@pytest.mark.parametrize("cap", [None, 32768])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("n", [1, 5, 40, 300])
@pytest.mark.parametrize("gap", [8, 16, 24])
def test_attend_sink(gap, n, f16, cap):
    """A first key that outweighs all others together and whose value is 0: the output is the others'.  Weights as two f16 parts
    are held to 2^-30 of the largest of their row: it is 2^6 or above; a small one's upper 11 bits and the rest become f16 numbers,
    each off by up to half a step of the least ones, 2^-25, so 2^-24 together.  Beside that the bounds of sums in f32, and 2^-22 or
    2^-39 of what a token sees for parts of keys and values."""
    b = Batch((8, 2, 128), f16, [n + 1000, n + 90, n + 1], [n] * 3, cap=cap, seed=gap + n, spread=0.15)
    sign = torch.where(torch.rand(128, generator=gen(gap), device="cuda") < 0.5, -7.0, 7.0)
    b.k *= 0.6
    b.k[:, :, 0], b.v[:, :, 0] = sign.to(b.k.dtype), 0
    b.q += sign * (gap / 49 / math.sqrt(128))
    want = b.expect()
    for r in range(3):
        v = b.v[r, :, : b.lens_h[r]].double().abs()
        upto = v.cumsum(1)[:, b.lens_h[r] - n :]  # [G][n][hd]: of the values that a token sees
        want[1][r] += (2.0**-30 * upto + 2.0**-38 * v.amax((1, 2), keepdim=True)).transpose(0, 1).repeat_interleave(4, 1)
    b.check(b.attend(), want)
    assert b.ops.errors(stream()) == 0
