"""The paged cache's operators against plain restatements in 64 bits, where they can go wrong: pages that end inside a tile,
lengths of zero and one, rows whose request or slot is none, strides and alignments, NaN and infinities in places that no row
may see, offsets past 32 bits."""
import numpy as np
import pytest
import torch

from ferrum_gpu_b200 import CudaError, PagedCache, RopeScaling, Rotary, Step, _ffi, rope_tables

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}  # half the distance of f16's smallest values


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype="f32", scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(DT[dtype])


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _sync(dev):
    torch.cuda.synchronize()
    dev.sync()
    torch.cuda.synchronize()


# ---- pages and slots ------------------------------------------------------------------------------------------------

class Book:
    """The plan's rules on the host."""

    def __init__(self, pages, page, requests, most, rng):
        self.page, self.most = page, most
        self.table = np.full((requests, most), -1, dtype=np.int32)
        self.lens = np.zeros(requests, dtype=np.int32)
        self.free = list(rng.permutation(pages).astype(np.int32))

    def pages(self, n):
        return -(-n // self.page)

    def extend(self, req, grow, rows):
        starts, out = [0], []
        need = sum(self.pages(self.lens[r] + g) - self.pages(self.lens[r]) for r, g in zip(req, grow))
        status = 0
        if any(self.lens[r] + g > self.most * self.page for r, g in zip(req, grow)):
            status = _ffi.FC_ERR_CONTEXT_FULL
        elif sum(grow) > rows:
            status = _ffi.FC_ERR_SHAPE
        elif need > len(self.free):
            status = need - len(self.free)
        for r, g in zip(req, grow) if not status else []:
            for p in range(self.pages(self.lens[r]), self.pages(self.lens[r] + g)):
                self.table[r, p] = self.free.pop()
            for pos in range(self.lens[r], self.lens[r] + g):
                out.append((int(self.table[r, pos // self.page]) * self.page + pos % self.page, pos, r))
            self.lens[r] += g
            starts.append(len(out))
        if status:
            starts = [0] * (len(req) + 1)
        out += [(-1, -1, -1)] * (rows - len(out))
        return starts, out, status

    def release(self, req):
        for r in req:
            self.free += list(self.table[r, :self.pages(self.lens[r])])
            self.lens[r] = 0


def _cache(dev, book, pages):
    free = np.full(pages, -7, dtype=np.int32)
    free[:len(book.free)] = book.free
    return PagedCache(dev, book.page, table=_i32(book.table), lens=_i32(book.lens), free=_i32(free), n_free=_i32([len(book.free)]))


def _same_book(dev, cache, book):
    _sync(dev)
    n = int(cache.n_free)
    assert n == len(book.free)
    np.testing.assert_array_equal(cache.free[:n].cpu().numpy(), book.free)
    np.testing.assert_array_equal(cache.table.cpu().numpy(), book.table)
    np.testing.assert_array_equal(cache.lens.cpu().numpy(), book.lens)


@pytest.mark.parametrize("page,requests,pages,most", [(1, 5, 300, 60), (16, 40, 700, 20), (256, 3, 30, 9), (8, 1500, 9000, 12), (2, 300, 200, 40)])
def test_a_life_of_steps_follows_the_rules(dev, page, requests, pages, most):
    rng = np.random.default_rng(page)
    book = Book(pages, page, requests, most, rng)
    cache = _cache(dev, book, pages)
    status = _i32([9])
    for turn in range(12):
        n = int(rng.integers(0, requests + 1))
        req = rng.permutation(requests)[:n]
        if turn % 4 == 3:
            cache.release(_i32(req), status)
            book.release(req)
            _sync(dev)
            assert int(status) == 0
        else:
            grow = rng.integers(0, 2 if turn % 2 else max(2, most * page // 6), size=n)
            rows = max(0, int(grow.sum()) + int(rng.integers(-2, 40)))
            step = Step.new(dev, n, rows)
            cache.extend(_i32(grow), step, requests=_i32(req))
            starts, out, want = book.extend(req.tolist(), grow.tolist(), rows)
            _sync(dev)
            assert int(step.status) == want
            assert step.starts.tolist() == starts
            got = list(zip(step.slot.tolist(), step.position.tolist(), step.request.tolist()))
            assert got == out
        _same_book(dev, cache, book)


def test_refused_steps_change_nothing(dev):
    book = Book(10, 4, 4, 5, np.random.default_rng(1))
    book.extend([0, 2], [5, 3], 100)
    cache = _cache(dev, book, 10)
    new_lens, new_free = _i32([-3] * 4), _i32([-3])
    for req, grow, rows, want in [([0, 1], [1, 40], 100, _ffi.FC_ERR_CONTEXT_FULL), ([0, 4], [1, 1], 100, _ffi.FC_ERR_RANGE),
                                  ([-1], [1], 100, _ffi.FC_ERR_RANGE), ([1], [-1], 100, _ffi.FC_ERR_RANGE), ([0, 1], [2, 2], 3, _ffi.FC_ERR_SHAPE),
                                  ([0, 1, 3], [15, 20, 16], 100, 5), ([1], [2 ** 31 - 1], 100, _ffi.FC_ERR_CONTEXT_FULL)]:
        step = Step.new(dev, len(req), rows)
        cache.extend(_i32(grow), step, requests=_i32(req), lens_out=new_lens, n_free_out=new_free)
        _sync(dev)
        assert int(step.status) == want, (req, grow)
        assert set(step.slot.tolist()) | set(step.position.tolist()) <= {-1} and set(step.starts.tolist()) == {0}
        _same_book(dev, cache, book)
        assert int(new_free) == len(book.free)
    for req, spoil, want in [([0, 9], None, _ffi.FC_ERR_RANGE), ([0, 2, 0, 2, 0, 2], None, _ffi.FC_ERR_SHAPE), ([2], (2, 0), _ffi.FC_ERR_RANGE)]:
        status = _i32([9])
        keep = cache.table.clone()
        if spoil:
            cache.table[spoil] = 10
        _sync(dev)
        cache.release(_i32(req), status)
        _sync(dev)
        assert int(status) == want, req
        cache.table.copy_(keep)
        _same_book(dev, cache, book)


def test_defaults_of_a_step(dev):
    """requests None is the first rows of the table; new lengths and stack height may go elsewhere; a step of nothing."""
    cache = PagedCache.new(dev, 0, 1, 8, pages=9, page=2, requests=3, max_pages=4, dtype=torch.float32)
    step, lens, left = Step.new(dev, 2, 4), _i32([7, 7, 7]), _i32([7])
    cache.extend(_i32([3, 1]), step, lens_out=lens, n_free_out=left)
    _sync(dev)
    assert step.starts.tolist() == [0, 3, 4] and step.position.tolist() == [0, 1, 2, 0] and step.request.tolist() == [0, 0, 0, 1]
    assert step.slot.tolist() == [0, 1, 2, 4] and lens.tolist() == [3, 1, 7] and int(left) == 6
    assert cache.lens.tolist() == [0, 0, 0] and int(cache.n_free) == 9
    empty = Step.new(dev, 0, 3)
    cache.extend(_i32([]), empty)
    _sync(dev)
    assert empty.starts.tolist() == [0] and empty.slot.tolist() == [-1] * 3 and int(empty.status) == 0
    only = Step(starts=_i32([1] * 3), status=_i32([1]))  # (no rows wanted)
    cache.extend(_i32([0, 0]), only)
    _sync(dev)
    assert only.starts.tolist() == [0, 0, 0] and int(only.status) == 0


# ---- rotary positions, k and v to their slots -------------------------------------------------------------------------

def _rotated(x, cos, sin, rope_dim, neox):
    """float64 [rows, heads, hd] rotated by the tables' rows."""
    out, half = x.clone(), rope_dim // 2
    i = torch.arange(half, device=x.device)
    a, b = (i, i + half) if neox else (2 * i, 2 * i + 1)
    c, s = cos.double()[:, None, :], sin.double()[:, None, :]
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., a] * s + x[..., b] * c
    return out


def _append_case(dev, rows, heads, kv, hd, rope_dim, neox, act, cache, page, positions=500, pad=0, shift=0, q_pad=0, q_shift=0, in_place=False, seed=0):
    g = _gen(seed)
    width = (heads + 2 * kv) * hd
    flat = _randn(g, rows * (width + pad) + shift, dtype=act)
    qkv = flat[shift:].view(rows, width + pad)[:, :width]
    n_pages = -(-rows // page) + 3
    k, v = (_randn(g, n_pages, kv, page, hd, dtype=cache) for _ in range(2))
    slot = torch.randperm(n_pages * page, device="cuda", generator=g)[:rows]
    position = torch.randint(0, positions, (rows,), device="cuda", generator=g).to(torch.int32)
    if rows > 3:
        slot[1], position[2], position[3] = -1, -1, positions  # no slot; no position; past the tables
    if rows > 4:
        slot[4] = n_pages * page  # past the pool
    want_k, want_v = k.double(), v.double()
    x = qkv.double().reshape(rows, heads + 2 * kv, hd)
    rotary = None
    if rope_dim:
        cos, sin = (torch.from_numpy(t).cuda() for t in rope_tables(RopeScaling(rope_dim, base=1e5), positions))
        rotary = Rotary(cos, sin, neox)
        at = position.long().clamp(0, positions - 1)
        x[:, :heads + kv] = _rotated(x[:, :heads + kv], cos[at], sin[at], rope_dim, neox)
    dead = (position < 0) | ((position >= positions) & bool(rope_dim))
    live = ~dead & (slot >= 0) & (slot < n_pages * page)
    want_k[slot[live] // page, :, slot[live] % page] = x[live, heads:heads + kv]
    want_v[slot[live] // page, :, slot[live] % page] = x[live, heads + kv:]
    want_q = torch.where(dead[:, None], 0.0, x[:, :heads].reshape(rows, -1))
    if in_place:
        q = qkv[:, :heads * hd]
    else:
        q = torch.full((rows * (heads * hd + q_pad) + q_shift,), 7.0, dtype=DT[act], device="cuda")[q_shift:].view(rows, -1)[:, :heads * hd]
    torch.cuda.synchronize()
    PagedCache(dev, page, layers=[(k, v)]).append(0, qkv, Step(slot=slot, position=position), q, rotary=rotary)
    _sync(dev)
    # f32: the product rounded, the fused sum rounded: 2 roundings of |a c| + |b s| <= sqrt(2) 6 (inputs of |x| < 6); then the type's rounding
    for got, want, kind in ((q.double(), want_q, act), (k.double(), want_k, cache), (v.double(), want_v, cache)):
        assert ((got - want).abs() <= 2 * 8.5 * 2.0 ** -24 + want.abs() * HALF_ULP[kind] * (1 + 2 ** -10) + TINY[kind]).all()
    untouched = torch.ones(n_pages * page, dtype=torch.bool, device="cuda")
    untouched[slot[live]] = False
    for got, want in ((k, want_k), (v, want_v)):
        a, b = (t.transpose(1, 2).reshape(n_pages * page, -1)[untouched] for t in (got.double(), want))
        assert torch.equal(a, b)


@pytest.mark.parametrize("act,cache", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f16")])
@pytest.mark.parametrize("neox", [False, True])
def test_append_types_and_layouts(dev, act, cache, neox):
    _append_case(dev, 37, 12, 4, 64, 64, neox, act, cache, 16, seed=1)
    _append_case(dev, 9, 4, 4, 128, 96, neox, act, cache, 8, seed=2)


@pytest.mark.parametrize("hd,rope_dim", [(8, 8), (8, 2), (24, 24), (40, 20), (64, 0), (64, 2), (64, 6), (72, 70), (80, 32), (128, 64), (200, 120), (256, 256)])
@pytest.mark.parametrize("neox", [False, True])
def test_append_head_sizes_and_parts_of_the_head(dev, hd, rope_dim, neox):
    _append_case(dev, 6, 3, 1, hd, rope_dim, neox, "f32", "f16", 4, seed=3)
    _append_case(dev, 5, 6, 3, hd, rope_dim, neox, "f16", "f16", 32, seed=4)


@pytest.mark.parametrize("rows,page", [(1, 1), (2, 256), (300, 2), (1000, 64)])
def test_append_rows_and_pages(dev, rows, page):
    _append_case(dev, rows, 16, 2, 64, 64, True, "f32", "f32", page, seed=5)


@pytest.mark.parametrize("kw", [dict(pad=8), dict(pad=1), dict(shift=1), dict(q_pad=3), dict(q_shift=1), dict(in_place=True), dict(in_place=True, pad=5, shift=3)])
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("neox", [False, True])
def test_append_strides_and_alignments(dev, kw, act, neox):
    _append_case(dev, 33, 6, 2, 64, 32, neox, act, "bf16" if act == "bf16" else "f32", 16, seed=6, **kw)


@pytest.mark.parametrize("act,cache", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("heads,kv,hd,rope_dim", [(12, 4, 64, 64), (32, 8, 128, 96), (3, 1, 40, 24), (64, 8, 128, 128), (6, 6, 64, 0), (56, 8, 256, 256), (2, 2, 64, 40)])
@pytest.mark.parametrize("neox", [False, True])
def test_append_many_rows(dev, act, cache, heads, kv, hd, rope_dim, neox):
    """Rows from narrow (a few hundred bytes) to wide (tens of KB), 20 MB of them; with rows that are no tokens."""
    _append_case(dev, 20_000_000 // ((heads + 2 * kv) * hd * (4 if act == "f32" else 2)), heads, kv, hd, rope_dim, neox, act, cache, 16, seed=7, pad=8 if heads == 12 else 0, q_pad=16 if heads == 6 else 0)


# ---- attention ----------------------------------------------------------------------------------------------------------

def _attend_case(dev, lens, heads, kv, hd, act, cache, page, scale=0.0, request=None, q_scale=2.0, seed=0, pad=0, shift=0, holes=(), n_pages=None, poison=True):
    """Rows of lengths `lens` (0: no position); request r by default, `request` where several rows share one."""
    g = _gen(seed)
    rows = len(lens)
    request = list(range(rows)) if request is None else request
    held = {}
    for r, n in zip(request, lens):
        held[r] = max(held.get(r, 0), -(-n // page))
    requests, most = max(request) + 2, max(max(held.values()), 1) + 1
    used = sum(held.values())
    n_pages = n_pages or used + 3
    order = torch.randperm(n_pages, device="cuda", generator=g)[:used].tolist()
    if n_pages > used:
        order = [n_pages - 1 - p if p < n_pages // 2 else p for p in order] if used == 1 else order
    table = torch.full((requests, most), -1, dtype=torch.int32, device="cuda")
    k, v = (torch.empty(n_pages, kv, page, hd, dtype=DT[cache], device="cuda") for _ in range(2))
    if poison:  # what nobody may see: NaN and infinities wherever no position was written
        k.fill_(float("nan"))
        v.fill_(float("inf"))
    for r, n in held.items():
        mine = [order.pop() for _ in range(n)]
        top = max(x for q, x in zip(request, lens) if q == r)
        for i, p in enumerate(mine):
            table[r, i] = p
            here = min(page, top - i * page)
            k[p, :, :here] = _randn(g, kv, here, hd, dtype=cache)
            v[p, :, :here] = _randn(g, kv, here, hd, dtype=cache)
    for r, i in holes:
        table[r, i] = n_pages + 5
    width = heads * hd
    q = _randn(g, rows * (width + pad) + shift, dtype=act, scale=q_scale)[shift:].view(rows, width + pad)[:, :width]
    out = torch.full((rows * (width + pad) + shift,), 7.0, dtype=DT[act], device="cuda")[shift:].view(rows, width + pad)[:, :width]
    step = Step(position=_i32([n - 1 for n in lens]), request=_i32(request))
    torch.cuda.synchronize()
    PagedCache(dev, page, table=table, layers=[(k, v)]).attend(0, q, step, out, scale=scale)
    _sync(dev)
    worst = 0.0
    for r in range(rows):
        n, req = lens[r], request[r]
        keep = [j for j in range(-(-n // page)) if (req, j) not in holes]
        got = out[r].double().view(heads, hd)
        if not keep:
            assert not got.any()
            continue
        pages = table[req, keep].long()
        ok = torch.cat([torch.arange(j * page, (j + 1) * page, device="cuda") for j in keep]) < n
        kk = k[pages].double().transpose(0, 1).reshape(kv, -1, hd)[:, ok]
        vv = v[pages].double().transpose(0, 1).reshape(kv, -1, hd)[:, ok]
        qq = q[r].double().view(kv, heads // kv, hd)
        f = scale or hd ** -0.5
        want = (torch.softmax(qq @ kk.transpose(1, 2) * f, dim=-1) @ vv).reshape(heads, hd)
        # A score's error: operands kept to 22 bits, their products summed in f32: 2^-20 of sum |q k| at most; a probability's
        # is twice that, its own terms and the sums' roundings are 2^-20 of it; then the result's type
        size = float((qq.abs() @ kk.abs().transpose(1, 2)).max()) * abs(f)
        tol = 2.0 ** -19 * (1 + size) * float(vv.abs().max()) + want.abs() * HALF_ULP[act] * (1 + 2 ** -10) + TINY[act]
        worst = max(worst, float(((got - want).abs() / tol).max()))
    assert worst <= 1.0, worst


TYPES = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f16")]


@pytest.mark.parametrize("act,cache", TYPES)
def test_attend_types(dev, act, cache):
    _attend_case(dev, [1, 700, 33, 0, 257], 12, 4, 64, act, cache, 16, seed=1)
    _attend_case(dev, [129, 5], 8, 1, 128, act, cache, 32, seed=2)


@pytest.mark.parametrize("page", [1, 2, 4, 8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("cache", ["f32", "f16"])
def test_attend_pages_and_lengths(dev, page, cache):
    _attend_case(dev, [1, 2, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513, 1000], 4, 2, 64, "f32", cache, page, seed=page)


@pytest.mark.parametrize("hd", [8, 16, 24, 32, 40, 56, 64, 72, 80, 96, 104, 112, 128, 136, 160, 192, 200, 248, 256])
@pytest.mark.parametrize("act,cache", [("f32", "f32"), ("f32", "bf16"), ("f16", "f16")])
def test_attend_head_sizes(dev, hd, act, cache):
    _attend_case(dev, [3, 70, 300], 6, 2, hd, act, cache, 16, seed=hd)


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 1), (5, 1), (8, 1), (9, 1), (16, 1), (17, 1), (71, 1), (6, 6), (24, 2), (64, 8), (40, 40)])
@pytest.mark.parametrize("cache", ["f32", "f16", "bf16"])
def test_attend_head_groupings(dev, heads, kv, cache):
    _attend_case(dev, [40, 1, 333], heads, kv, 64, "f32", cache, 16, seed=heads)


def test_attend_rows_that_see_nothing(dev):
    _attend_case(dev, [0, 0, 5, 0], 4, 2, 64, "f32", "f16", 16, seed=1)
    _attend_case(dev, [0], 4, 2, 64, "f16", "f16", 16, seed=2)
    _attend_case(dev, [40, 17, 0, 33], 4, 2, 64, "f32", "f32", 16, holes=[(0, 1), (1, 0), (1, 1), (3, 2)], seed=3)
    _attend_case(dev, [200, 17], 4, 2, 64, "bf16", "bf16", 4, holes=[(0, 3), (0, 49), (1, 0)], seed=4)
    # requests and positions that are none: 0, and the table is not read outside
    cache = PagedCache(dev, 8, table=_i32([[0, 1], [-1, -1]]), layers=[(torch.ones(2, 1, 8, 64, device="cuda"), torch.ones(2, 1, 8, 64, device="cuda"))])
    q, out = torch.ones(6, 64, device="cuda"), torch.full((6, 64), 7.0, device="cuda")
    step = Step(position=_i32([15, 3, 3, -5, 2 ** 31 - 1, 3]), request=_i32([0, -1, 2, 0, 0, 1]))
    torch.cuda.synchronize()
    cache.attend(0, q, step, out)
    _sync(dev)
    assert torch.equal(out, _i32([1, 0, 0, 0, 1, 0])[:, None].float().expand(6, 64))


def test_attend_rows_of_one_request_see_their_own_past(dev):
    """A prompt's rows: causal, each up to its own position."""
    _attend_case(dev, list(range(1, 50)), 8, 2, 64, "f32", "f16", 16, request=[1] * 49, seed=1)
    _attend_case(dev, [5, 300, 301, 7, 302, 0], 6, 3, 128, "f32", "f32", 64, request=[2, 0, 0, 2, 0, 1], seed=2)


@pytest.mark.parametrize("cache", ["f32", "f16", "bf16"])
def test_attend_long_and_uneven(dev, cache):
    _attend_case(dev, [20001], 16, 2, 64, "f32", cache, 64, seed=1)
    _attend_case(dev, [9000, 1, 1, 3000, 17, 1, 1, 1, 1], 8, 8, 128, "f32", cache, 16, seed=2)
    _attend_case(dev, [1 + (i * 37) % 90 for i in range(200)], 4, 2, 64, "f32", cache, 16, seed=3)


@pytest.mark.parametrize("kw", [dict(pad=3), dict(shift=1), dict(pad=8, shift=8), dict(scale=1.0), dict(scale=-0.3), dict(q_scale=40.0), dict(q_scale=1e-6), dict(q_scale=1e-3)])
@pytest.mark.parametrize("act,cache", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
def test_attend_strides_scales_and_sizes(dev, kw, act, cache):
    _attend_case(dev, [300, 41], 8, 2, 64, act, cache, 16, seed=7, **kw)


@pytest.mark.parametrize("cache", ["f32", "f16"])
def test_attend_large_queries_and_small_keys_keep_their_bits(dev, cache):
    """q of 10^6 against k of 10^-6 (f16: 10^-3): the products are ordinary."""
    g = _gen(3)
    n, hd, small = 77, 64, 1e-6 if cache == "f32" else 1e-3
    k, v = _randn(g, 5, 1, 16, hd, dtype=cache, scale=small), _randn(g, 5, 1, 16, hd, dtype=cache)
    q = _randn(g, 1, 4 * hd, scale=1 / small)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    PagedCache(dev, 16, table=_i32([[3, 1, 0, 2, 4]]), layers=[(k, v)]).attend(0, q, Step(position=_i32([n - 1])), out)
    _sync(dev)
    kk, vv = (t[[3, 1, 0, 2, 4], 0].reshape(-1, hd)[:n].double() for t in (k, v))
    want = torch.softmax(q.double().view(4, hd) @ kk.T / 8, dim=-1) @ vv
    size = float((q.double().view(4, hd).abs() @ kk.abs().T).max()) / 8
    assert float((out.double().view(4, hd) - want).abs().max()) <= 2.0 ** -19 * (1 + size) * float(vv.abs().max())


def test_attend_offsets_past_32_bits(dev):
    """The last pages of a pool of 4.5 G elements (f16) and 1.2 G (f32: past 2^32 bytes)."""
    for cache, n_pages in (("f16", 4_500_000), ("f32", 1_200_000)):
        _attend_case(dev, [60], 4, 1, 64, "f32", cache, 16, n_pages=n_pages, seed=1, poison=False)
        _attend_case(dev, [9], 4, 1, 64, "f32", cache, 16, n_pages=n_pages, seed=2, poison=False)
        torch.cuda.empty_cache()


def test_append_offsets_past_32_bits(dev):
    n_pages, page, hd = 4_500_000, 16, 64
    k, v = (torch.empty(n_pages, 1, page, hd, dtype=torch.float16, device="cuda") for _ in range(2))
    slot = torch.tensor([n_pages * page - 1, n_pages * page - 17, 5], device="cuda")
    qkv = _randn(_gen(1), 3, 3 * hd, dtype="f16")
    q = torch.empty(3, hd, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    PagedCache(dev, page, layers=[(k, v)]).append(0, qkv, Step(slot=slot, position=_i32([0, 1, 2])), q)
    _sync(dev)
    for r, s in enumerate(slot.tolist()):
        assert torch.equal(k[s // page, 0, s % page], qkv[r, hd:2 * hd]) and torch.equal(v[s // page, 0, s % page], qkv[r, 2 * hd:])
    del k, v
    torch.cuda.empty_cache()


def test_a_captured_step_replays_with_new_lengths(dev):
    """extend, append and attend in one graph of a fixed shape: replays see the lengths of their own turn."""
    page, kv, heads, hd, rows = 16, 2, 4, 64, 5
    cache = PagedCache.new(dev, 1, kv, hd, pages=40, page=page, requests=4, max_pages=6, dtype=torch.float32)
    rotary = Rotary.build(dev, RopeScaling(hd), 100, True)
    step, grow = Step.new(dev, 4, rows), _i32([1, 0, 1, 1])
    qkv = torch.zeros(rows, (heads + 2 * kv) * hd, device="cuda")
    q, out = (torch.zeros(rows, heads * hd, device="cuda") for _ in range(2))
    torch.cuda.synchronize()

    def call():
        cache.extend(grow, step)
        cache.append(0, qkv, step, q, rotary=rotary)
        cache.attend(0, q, step, out)

    graph = torch.cuda.CUDAGraph()
    stream = dev.torch_stream()
    with torch.cuda.stream(stream):
        graph.capture_begin(capture_error_mode="thread_local")
        call()
        graph.capture_end()
    history = {0: [], 2: [], 3: []}
    cos, sin = (t.double() for t in (rotary.cos, rotary.sin))
    for turn in range(20):
        qkv.copy_(_randn(_gen(turn), rows, (heads + 2 * kv) * hd))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        _sync(dev)
        assert step.request.tolist() == [0, 2, 3, -1, -1] and step.position.tolist() == [turn] * 3 + [-1, -1] and int(step.status) == 0
        x = qkv.double().view(rows, heads + 2 * kv, hd)
        x = torch.cat([_rotated(x[:, :heads + kv], cos[[turn] * rows], sin[[turn] * rows], hd, True), x[:, heads + kv:]], dim=1)
        for r, req in enumerate((0, 2, 3)):
            history[req].append(x[r, heads:])
            kv_all = torch.stack(history[req])
            kk, vv = kv_all[:, :kv].transpose(0, 1), kv_all[:, kv:].transpose(0, 1)
            want = torch.softmax(x[r, :heads].view(kv, heads // kv, hd) @ kk.transpose(1, 2) / 8, dim=-1) @ vv
            assert float((out[r].double().view(kv, heads // kv, hd) - want).abs().max()) < 1e-4
        assert not out[3:].any()

def test_attend_table_limits(dev):
    """A call's tiles are counted in 32 bits: wide page tables under many rows are taken as far as that goes, and refused behind it."""
    f = torch.zeros
    pool = f(1, 1, 256, 8, device="cuda") + 1
    table = f(1, 1 << 20, dtype=torch.int32, device="cuda")  # 2^28 positions: 2^22 tiles of 64
    cache = PagedCache(dev, 256, table=table, layers=[(pool, pool)])

    def call(rows):
        q, out = f(rows, 32, device="cuda"), f(rows, 32, device="cuda")
        step = Step(position=f(rows, dtype=torch.int32, device="cuda") + 2, request=f(rows, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        cache.attend(0, q, step, out)
        _sync(dev)
        return out

    assert (call(1000) == 1).all()
    with pytest.raises(CudaError, match="more than one call holds") as e:
        call(1025)
    assert e.value.code == _ffi.FC_ERR_UNSUPPORTED



def test_results_do_not_change_from_call_to_call(dev):
    g = _gen(5)
    k, v = (_randn(g, 300, 2, 16, 64, dtype="f16") for _ in range(2))
    table = torch.randperm(300, device="cuda", generator=g).to(torch.int32).view(3, 100)
    q = _randn(g, 3, 8 * 64)
    cache, step = PagedCache(dev, 16, table=table, layers=[(k, v)]), Step(position=_i32([1599, 900, 1234]))
    outs = [torch.empty_like(q) for _ in range(20)]
    torch.cuda.synchronize()
    for out in outs:
        cache.attend(0, q, step, out)
    _sync(dev)
    assert all(torch.equal(out, outs[0]) for out in outs)


# ---- refusals -------------------------------------------------------------------------------------------------------------

def test_refusals(dev):
    f = torch.zeros
    kv = [(f(4, 2, 16, 64, device="cuda"), f(4, 2, 16, 64, device="cuda"))]
    table = f(3, 4, dtype=torch.int32, device="cuda")
    cache = PagedCache(dev, 16, table=table, layers=kv)
    step = Step(slot=f(5, dtype=torch.int64, device="cuda"), position=f(5, dtype=torch.int32, device="cuda"), request=f(5, dtype=torch.int32, device="cuda"))
    q = f(5, 256, device="cuda")
    out = f(5, 256, device="cuda")

    def refused(code, match, call, *a, **kw):
        with pytest.raises(CudaError, match=match) as e:
            call(*a, **kw)
        assert e.value.code == code

    A, S, U, R = _ffi.FC_ERR_ARG, _ffi.FC_ERR_SHAPE, _ffi.FC_ERR_UNSUPPORTED, _ffi.FC_ERR_RANGE
    refused(U, "power of two", PagedCache(dev, 24, table=table, layers=[(f(4, 2, 24, 64, device="cuda"),) * 2]).attend, 0, q, step, out)
    refused(U, "multiple of 8", PagedCache(dev, 16, table=table, layers=[(f(4, 2, 16, 60, device="cuda"),) * 2]).attend, 0, f(5, 240, device="cuda"), step, f(5, 240, device="cuda"))
    refused(U, "multiple of 8", PagedCache(dev, 16, table=table, layers=[(f(4, 1, 16, 264, device="cuda"),) * 2]).attend, 0, f(5, 264, device="cuda"), step, f(5, 264, device="cuda"))
    refused(S, "not a multiple of kv_heads", cache.attend, 0, f(5, 192, device="cuda"), step, f(5, 192, device="cuda"))
    refused(S, "no whole heads", cache.attend, 0, f(5, 200, device="cuda"), step, f(5, 200, device="cuda"))
    refused(S, "q's shape and type", cache.attend, 0, q, step, f(5, 256, dtype=torch.float16, device="cuda"))
    refused(U, "float32, float16 or bfloat16", cache.attend, 0, q.double(), step, out.double())
    refused(A, "side by side", cache.attend, 0, f(256, 5, device="cuda").T, step, out)
    refused(S, "needs 6", cache.attend, 0, f(6, 256, device="cuda"), step, f(6, 256, device="cuda"))
    refused(A, "not finite", cache.attend, 0, q, step, out, scale=float("inf"))
    refused(R, "5 rows in a table of 3", cache.attend, 0, q, Step(position=step.position), out)
    refused(A, "page table", PagedCache(dev, 16, layers=kv).attend, 0, q, step, out)
    refused(R, "layer 1 of 1", cache.attend, 1, q, step, out)
    refused(A, "contiguous torch.int32", Step, position=step.position.long(), request=step.request)
    refused(A, "on cuda", cache.attend, 0, q.cpu(), step, out)
    qkv = f(5, 512, device="cuda")
    refused(S, "q_out must be", cache.append, 0, qkv, step, f(5, 255, device="cuda"))
    refused(A, "a pointer is NULL", cache.append, 0, qkv, Step(position=step.position), out)
    refused(S, "rope_dim 66", cache.append, 0, qkv, step, out, rotary=Rotary(f(9, 33, device="cuda"), f(9, 33, device="cuda"), True))
    refused(S, "hold no whole heads", cache.append, 0, f(5, 250, device="cuda"), step, out)
    refused(A, "cos must|sin must", Rotary, f(9, 32, device="cuda"), f(9, 31, device="cuda"), True)
    refused(A, "contiguous", PagedCache, dev, 16, layers=[(f(4, 2, 64, 16, device="cuda").transpose(2, 3),) * 2])
    refused(S, "one shape and type", PagedCache, dev, 16, layers=[(kv[0][0], kv[0][1].half())])
    full = PagedCache.new(dev, 0, 1, 8, pages=9, page=2, requests=3, max_pages=4, dtype=torch.float32)
    grow = _i32([1, 1])
    refused(A, "starts is NULL", full.extend, grow, Step(status=_i32([0])))
    refused(A, "status word", full.extend, grow, Step(starts=_i32([0] * 3)))
    refused(S, "needs 3", full.extend, grow, Step(starts=_i32([0] * 2), status=_i32([0])))
    refused(S, "one length", full.extend, grow, Step(starts=_i32([0] * 3), slot=f(4, dtype=torch.int64, device="cuda"), position=_i32([0] * 3), status=_i32([0])))
    refused(R, "4 requests in a table of 3", full.extend, _i32([1] * 4), Step(starts=_i32([0] * 5), status=_i32([0])))
    refused(U, "at most 8192 requests", full.release, _i32([0] * 8193), _i32([0]))
    refused(A, "status word", full.release, _i32([0]), None)
    refused(A, "needs the table", cache.release, _i32([0]), _i32([0]))
    # a refused launch (the host's fault hook) is reported and leaves the handle usable
    dev.fail_after(0)
    refused(_ffi.FC_ERR_INJECTED, "injected", cache.attend, 0, q, step, out)
    dev.fail_after(None)
    cache.attend(0, q, step, out)
    _sync(dev)
