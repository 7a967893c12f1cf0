"""8-bit pools (kv_dtype "e4m3"): the quantising append and its read-back bit
for bit, attention over quantised pages against 64 bits, forks and copies,
masked NaN, captured steps and the calls that are refused."""

import ctypes
import math
import random

import pytest

from flint_amd import ThubanError, _lib, ops
from flint_amd.pool import ArenaSpec, KvPool, RowMeta
from flint_amd.rope import Rope, rope_rows
from tests import q8_util
from tests.gpu_util import make_pool, scattered_alloc

pytestmark = pytest.mark.gpu


def _dt(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _load(torch, pool, rows, m, dt, layer=0, row_off=0):
    hd = pool.layer_info(layer).head_dim
    k, v = (torch.full((m, pool.kv_heads, hd), 7.0, dtype=dt, device="cuda") for _ in range(2))
    ops.kv_load(k, v, pool, layer, m, rows, row_off)
    return k, v


def _same(a, b):
    """Equal values, NaN equal to NaN."""
    return ((a == b) | (a.isnan() & b.isnan())).all().item()


def _kv(torch, g, n, nkv, hd, dt):
    chan = torch.exp2(torch.randn(nkv, hd, device="cuda", generator=g))
    k = torch.randn(n, nkv, hd, device="cuda", generator=g) * chan * 0.5
    v = torch.randn(n, nkv, hd, device="cuda", generator=g) * torch.exp2(
        torch.randn(n, nkv, 1, device="cuda", generator=g))
    return k.to(dt), v.to(dt)


class Filled:
    """A pool whose sequences hold `lens` tokens on scattered pages, and their
    stored values (k[s], v[s]: [n, kv_heads, hd], f64)."""

    def __init__(self, torch, lens, nkv, hd, page=16, seed=0, src="f32", budget=None, part_len=0, extra=3, layers=1):
        rng = random.Random(seed)
        self.torch, self.nkv, self.hd = torch, nkv, hd
        self.pool = make_pool(lens, nkv, hd, page_len=page, kv_dtype="e4m3", seq_lens=budget or lens,
                              extra_pages=extra, part_len=part_len, layers=layers)
        scattered_alloc(self.pool, lens, rng, page)
        self.k, self.v = [], []
        g = torch.Generator(device="cuda").manual_seed(seed)
        rows = RowMeta(max(max(lens), 1))
        for s, n in enumerate(lens):
            k, v = _kv(torch, g, n, nkv, hd, _dt(torch, src))
            if n:
                rows.write(list(range(n)), [s] * n)
                ops.kv_store(k, v, self.pool, 0, n, rows)
            self.k.append(q8_util.stored(k))
            self.v.append(q8_util.stored(v))
        torch.cuda.synchronize()
        self.g = g

    def query(self, m, nq, dt):
        return (self.torch.randn(m, nq, self.hd, device="cuda", generator=self.g) * 1.5).to(dt)

    def want(self, q, chunks, window, softcap, causal=True):
        """y and bound of rows of `chunks`: (sequence, positions)."""
        ys, bs, at = [], [], 0
        for s, pos in chunks:
            y, b = q8_util.attend(q[at:at + len(pos)], self.k[s], self.v[s], q8_util.row_ranges(pos, window, causal),
                                  1 / math.sqrt(self.hd), softcap)
            ys.append(y)
            bs.append(b)
            at += len(pos)
        return self.torch.cat(ys), self.torch.cat(bs)


def _spec(chunks, nq, hd, window=0, softcap=0.0, causal=True, seq=None):
    pos = [p for _, ps in chunks for p in ps]
    owner = [s for s, ps in chunks for _ in ps]
    rows = RowMeta(len(pos))
    rows.write(pos, owner)
    return ops.AttnSpec(q_heads=nq, window=window, scale=1 / math.sqrt(hd), m=len(pos), causal=causal, seq=seq,
                        args=rows, softcap=softcap)


# ------------------------------------------------------- append and read-back


@pytest.mark.parametrize("nkv,hd,page,m", [(8, 128, 16, 37), (2, 64, 32, 130), (3, 72, 16, 5), (1, 512, 64, 9),
                                           (4, 256, 256, 300), (5, 200, 16, 1), (4, 96, 32, 4099)])
@pytest.mark.parametrize("src,dst", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f16", "f32")])
def test_append_and_read_back(torch_cuda, nkv, hd, page, m, src, dst):
    torch = torch_cuda
    pool = make_pool([m + 40], nkv, hd, page_len=page, kv_dtype="e4m3", extra_pages=2)
    scattered_alloc(pool, [m + 40], random.Random(hd), page)
    g = torch.Generator(device="cuda").manual_seed(m)
    first = 23 if m < 4000 else 7
    rows = RowMeta(m)
    rows.write(list(range(first, first + m)), [0] * m)
    k, v = _kv(torch, g, m, nkv, hd, _dt(torch, src))
    ops.kv_store(k, v, pool, 0, m, rows)
    lk, lv = _load(torch, pool, rows, m, _dt(torch, dst))
    for x, y in ((k, lk), (v, lv)):
        assert _same(q8_util.stored(x).to(_dt(torch, dst)), y)
    # stored again from what was read back: the same values
    k32, v32 = _load(torch, pool, rows, m, torch.float32)
    ops.kv_store(k32, v32, pool, 0, m, rows)
    k2, v2 = _load(torch, pool, rows, m, torch.float32)
    assert _same(k32, k2) and _same(v32, v2)


def test_special_vectors(torch_cuda):
    """Zeros, ties between codes, the 448 border, subnormals, the largest
    floats, infinities and NaN (each alone in its vector)."""
    torch = torch_cuda
    hd = 64
    pool = make_pool([64], 1, hd, kv_dtype="e4m3")
    pool.alloc(0, 0, 64)
    x = torch.zeros(32, 1, hd, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(5)
    x[1, 0, 3] = 448.0 * 2 ** -9
    x[2, 0, 3] = 448.00003  # the next f32
    x[3, 0] = torch.arange(hd, device="cuda") * 0.0625 * 17  # ties of 5-bit significands
    x[4, 0] = torch.arange(hd, device="cuda") * 2.0 ** -10
    x[4, 0, 0] = 448.0  # subnormal codes and their ties under the largest scale
    x[5, 0] = torch.randn(hd, device="cuda", generator=g) * 1e-40
    x[6, 0] = torch.randn(hd, device="cuda", generator=g) * 1e38
    x[7, 0] = 3.4028234e38
    x[8, 0, 7] = math.inf
    x[9, 0, 8] = -math.inf
    x[10, 0, 9] = math.nan
    x[11, 0] = -0.0
    x[12, 0] = 1.1754944e-38
    x[13, 0] = 464.0
    x[14, 0] = 479.0
    x[15:, 0] = torch.randn(17, hd, device="cuda", generator=g).exp2() * torch.exp2(
        torch.randn(17, 1, device="cuda", generator=g) * 30)
    rows = RowMeta(32)
    rows.write(list(range(3, 35)), [0] * 32)
    ops.kv_store(x, x.flip(0).contiguous(), pool, 0, 32, rows)
    want = q8_util.stored(x)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        k, v = _load(torch, pool, rows, 32, dt)
        # (f64 to f32 is exact here; f32 to the 16-bit type is the one rounding)
        assert _same(want.float().to(dt), k) and _same(want.flip(0).float().to(dt), v)


def test_read_back_leaves_other_rows(torch_cuda):
    """Rows before and behind a call's keep what they hold, in the pool and in the destination."""
    torch = torch_cuda
    f = Filled(torch, [70, 33], 2, 128)
    rows = RowMeta(8)
    rows.write([5, 6, 7, 9, 32, 5, 5, 0], [0, 0, 0, 0, 1, 1, 0, 1])  # a token may be read twice
    k, v = (torch.full((10, 2, 128), 7.0, device="cuda") for _ in range(2))
    ops.kv_load(k[1:], v[1:], f.pool, 0, 7, rows, 1)
    for i, (s, p) in enumerate([(0, 6), (0, 7), (0, 9), (1, 32), (1, 5), (0, 5), (1, 0)]):
        assert _same(k[1 + i].double(), f.k[s][p]) and _same(v[1 + i].double(), f.v[s][p])
    assert (k[0] == 7).all() and (k[8:] == 7).all() and (v[0] == 7).all() and (v[8:] == 7).all()
    # append three tokens in the middle of a group of four: the others stay
    g = torch.Generator(device="cuda").manual_seed(9)
    nk, nv = _kv(torch, g, 3, 2, 128, torch.float16)
    rows.write([17, 18, 21], [0] * 3)
    ops.kv_store(nk, nv, f.pool, 0, 3, rows)
    f.k[0][[17, 18, 21]], f.v[0][[17, 18, 21]] = q8_util.stored(nk), q8_util.stored(nv)
    rows = RowMeta(70)
    rows.write(list(range(70)), [0] * 70)
    k, v = _load(torch, f.pool, rows, 70, torch.float32)
    assert _same(k.double(), f.k[0]) and _same(v.double(), f.v[0])


# ------------------------------------------------------------------ attention

DECODE = [
    # nq, nkv, hd, page, lens, q, y, window, softcap, part_len
    (14, 2, 64, 16, [1, 2, 15, 16, 17, 130, 511], "f32", "f32", 0, 0.0, 0),
    (32, 8, 128, 16, [1, 33, 900, 2500], "f16", "f16", 0, 0.0, 0),
    (40, 8, 128, 32, [5000, 63, 4097], "bf16", "bf16", 0, 0.0, 0),
    (16, 8, 256, 16, [700, 1, 95], "f32", "f32", 0, 50.0, 0),
    (8, 8, 512, 64, [333, 16, 77], "f16", "f32", 0, 0.0, 0),
    (4, 2, 512, 16, [200, 3], "f32", "f32", 0, 0.0, 64),
    (20, 1, 128, 16, [1000, 31], "f32", "bf16", 0, 0.0, 256),   # 20 query heads a KV head: two groups
    (12, 4, 96, 64, [20, 641], "f16", "f32", 0, 0.0, 0),
    (9, 3, 80, 16, [100, 257], "bf16", "f32", 50, 0.0, 0),
    (6, 3, 72, 256, [600, 10], "f32", "f16", 1, 0.0, 0),
    (5, 5, 192, 32, [300], "f16", "f16", 33, 20.0, 128),
    (7, 1, 320, 16, [90, 400], "f32", "f32", 0, 0.0, 128),
]


@pytest.mark.parametrize("nq,nkv,hd,page,lens,qd,yd,window,cap,part", DECODE)
def test_decode(torch_cuda, nq, nkv, hd, page, lens, qd, yd, window, cap, part):
    torch = torch_cuda
    f = Filled(torch, lens, nkv, hd, page, seed=hd + nq, part_len=part)
    chunks = [(s, [n - 1]) for s, n in enumerate(lens)]
    spec = _spec(chunks, nq, hd, window, cap)
    q = f.query(len(lens), nq, _dt(torch, qd))
    y = torch.zeros(len(lens), nq, hd, dtype=_dt(torch, yd), device="cuda")
    ops.attn(q, f.pool, 0, y, spec)
    want, bound = f.want(q, chunks, window, cap)
    q8_util.check(f"decode {nq}/{nkv}x{hd}", y, want, bound, y.dtype)
    # the no-allocation call (merge kernel) gives the same bits
    y2 = torch.zeros_like(y)
    c = ops._spec_c(spec, q, y2)
    _lib.check(_lib.lib().thb_attn_noalloc(f.pool.handle, 0, q.data_ptr(), y2.data_ptr(), ctypes.byref(c),
                                           spec.args.handle, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(y, y2)


CHUNKS = [
    # nq, nkv, hd, page, [(tokens, new)], q, y, window, softcap, part_len
    (32, 8, 128, 16, [(300, 300)], "f16", "f16", 0, 0.0, 0),
    (14, 2, 64, 32, [(777, 130), (64, 64), (5, 1)], "f32", "f32", 0, 0.0, 256),
    (16, 8, 256, 16, [(1001, 77), (900, 4), (900, 4)], "f32", "f32", 300, 50.0, 0),
    (40, 8, 128, 64, [(61, 61), (2000, 1), (1000, 129)], "bf16", "bf16", 0, 0.0, 0),
    (12, 4, 96, 16, [(500, 61)], "f16", "f32", 0, 0.0, 128),
    (9, 3, 80, 16, [(200, 200)], "f32", "f32", 17, 0.0, 0),
    (20, 1, 128, 16, [(90, 33)], "f16", "f32", 0, 0.0, 0),
    (4, 2, 512, 32, [(150, 65)], "f16", "f32", 0, 0.0, 64),
    (8, 8, 128, 16, [(1025, 1025)], "f16", "f32", 0, 0.0, 512),
]


@pytest.mark.parametrize("nq,nkv,hd,page,seqs,qd,yd,window,cap,part", CHUNKS)
def test_chunks(torch_cuda, nq, nkv, hd, page, seqs, qd, yd, window, cap, part):
    torch = torch_cuda
    f = Filled(torch, [n for n, _ in seqs], nkv, hd, page, seed=hd, part_len=part, src="bf16")
    chunks = [(s, list(range(n - new, n))) for s, (n, new) in enumerate(seqs)]
    spec = _spec(chunks, nq, hd, window, cap)
    q = f.query(spec.m, nq, _dt(torch, qd))
    y = torch.zeros(spec.m, nq, hd, dtype=_dt(torch, yd), device="cuda")
    ops.attn(q, f.pool, 0, y, spec)
    want, bound = f.want(q, chunks, window, cap)
    q8_util.check(f"chunks {nq}/{nkv}x{hd}", y, want, bound, y.dtype)


def test_fixed_sequence_and_not_causal(torch_cuda):
    """The reference's call of one sequence, without the causal mask, and rows in falling order."""
    torch = torch_cuda
    f = Filled(torch, [50, 400], 2, 64)
    for causal, pos in ((False, [10, 399]), (True, [399, 20, 5]), (True, [3])):
        spec = _spec([(1, pos)], 8, 64, causal=causal, seq=1)
        q = f.query(len(pos), 8, torch.float32)
        y = torch.zeros_like(q)
        ops.attn(q, f.pool, 0, y, spec)
        want, bound = f.want(q, [(1, pos)], 0, 0.0, causal)
        q8_util.check(f"fixed sequence causal={causal} {pos}", y, want, bound, y.dtype)


def test_large_and_small_magnitudes(torch_cuda):
    """Scales far from 1 stay out of the 16-bit operands."""
    torch = torch_cuda
    for ks, vs, qs in ((1e-12, 1e20, 1e12), (1e12, 1e-20, 1e-12), (1e6, 1e-30, 1e-6)):
        pool = make_pool([300], 2, 128, kv_dtype="e4m3")
        pool.alloc(0, 0, 300)
        g = torch.Generator(device="cuda").manual_seed(3)
        k, v = _kv(torch, g, 300, 2, 128, torch.float32)
        k, v = k * ks, v * vs
        rows = RowMeta(300)
        rows.write(list(range(300)), [0] * 300)
        ops.kv_store(k, v, pool, 0, 300, rows)
        pos = [299]
        spec = _spec([(0, pos)], 8, 128)
        q = torch.randn(1, 8, 128, device="cuda", generator=g) * qs
        y = torch.zeros_like(q)
        ops.attn(q, pool, 0, y, spec)
        want, bound = q8_util.attend(q, q8_util.stored(k), q8_util.stored(v), [(0, 300)], 1 / math.sqrt(128))
        q8_util.check(f"scales {ks} {vs} {qs}", y, want, bound, y.dtype)


@pytest.mark.parametrize("hd,new", [(64, 4), (128, 4), (128, 70), (256, 3)])
def test_masked_nan(torch_cuda, hd, new):
    """A NaN token reaches the rows that read it and no other: not the rows
    before it in the same chunk, not through slots of reused pages."""
    torch = torch_cuda
    n = 160
    f = Filled(torch, [n], 2, hd, budget=[n + 64])
    rows = RowMeta(256)
    pos = list(range(n - new, n))
    bad = n - new + new // 2
    rows.write([bad], [0])
    x = torch.full((1, 2, hd), math.nan, device="cuda")
    z = torch.ones(1, 2, hd, device="cuda")
    for k, v in ((x, z), (z, x)):
        ops.kv_store(k, v, f.pool, 0, 1, rows)
        f.k[0][bad], f.v[0][bad] = q8_util.stored(k)[0], q8_util.stored(v)[0]
        spec = _spec([(0, pos)], 8, hd)
        q = f.query(new, 8, torch.float16)
        y = torch.zeros(new, 8, hd, device="cuda")
        ops.attn(q, f.pool, 0, y, spec)
        first = next(i for i, p in enumerate(pos) if p >= bad)
        assert y[first:].isnan().all() and not y[:first].isnan().any()
        want, bound = f.want(q[:first], [(0, pos[:first])], 0, 0.0)
        q8_util.check("rows before the NaN", y[:first], want, bound, y.dtype)


def test_stale_nan_pages(torch_cuda):
    torch = torch_cuda
    pool = KvPool(ArenaSpec([64, 64], 4), 2, 128, page_len=32, kv_dtype="e4m3")
    pool.alloc(0, 0, 64)
    pool.alloc(1, 0, 64)
    rows = RowMeta(128)
    rows.write(list(range(64)) * 2, [0] * 64 + [1] * 64)
    x = torch.full((128, 2, 128), math.nan, device="cuda")
    ops.kv_store(x, x, pool, 0, 128, rows)
    pool.free_seq(0)
    pool.free_seq(1)
    g = torch.Generator(device="cuda").manual_seed(1)
    for n in (1, 3, 17, 31, 33, 50):
        pool.alloc(0, 0, n)
        k, v = _kv(torch, g, n, 2, 128, torch.float32)
        rows.write(list(range(n)), [0] * n)
        ops.kv_store(k, v, pool, 0, n, rows)
        spec = _spec([(0, [n - 1])], 8, 128)
        q = torch.randn(1, 8, 128, device="cuda", generator=g)
        y = torch.zeros_like(q)
        ops.attn(q, pool, 0, y, spec)
        want, bound = q8_util.attend(q, q8_util.stored(k), q8_util.stored(v), [(0, n)], 1 / math.sqrt(128))
        q8_util.check(f"{n} tokens on stale pages", y, want, bound, y.dtype)
        pool.free_seq(0)
        pool.alloc(1, 0, 64)
        rows.write(list(range(64)), [1] * 64)
        ops.kv_store(x[:64], x[:64], pool, 0, 64, rows)
        pool.free_seq(1)


def test_batch_equals_solo_and_placement(torch_cuda):
    """A row's bits depend neither on the other rows nor on where its pages are."""
    torch = torch_cuda
    lens = [1500, 40, 4500, 700]
    a = Filled(torch, lens, 8, 128, seed=4)
    q = a.query(len(lens), 32, torch.float16)
    y = torch.zeros(len(lens), 32, 128, device="cuda")
    ops.attn(q, a.pool, 0, y, _spec([(s, [n - 1]) for s, n in enumerate(lens)], 32, 128))
    b = Filled(torch, lens, 8, 128, seed=4, extra=40)
    for s, n in enumerate(lens):
        z = torch.zeros(1, 32, 128, device="cuda")
        ops.attn(q[s:s + 1].contiguous(), b.pool, 0, z, _spec([(s, [n - 1])], 32, 128))
        assert torch.equal(z[0], y[s])
    again = torch.zeros_like(y)
    ops.attn(q, a.pool, 0, again, _spec([(s, [n - 1]) for s, n in enumerate(lens)], 32, 128))
    assert torch.equal(again, y)


# --------------------------------------------------- the page API and copies


@pytest.mark.parametrize("hd,page", [(64, 16), (96, 32), (128, 16), (256, 64)])
def test_fork_truncate_copy(torch_cuda, hd, page):
    torch = torch_cuda
    n = 5 * page + 7
    f = Filled(torch, [n], 3, hd, page, budget=[n + 40, n + 40, n + 40], extra=12)
    f.pool.fork(0, 1, n)
    f.pool.fork(0, 2, 2 * page + 5)
    g = torch.Generator(device="cuda").manual_seed(8)
    rows = RowMeta(200)
    k0, v0 = f.k[0].clone(), f.v[0].clone()
    # both forks and the source append different tokens; a shared page is copied first
    held = {0: n, 1: n, 2: 2 * page + 5}
    f.k, f.v = [k0, k0.clone(), k0[:held[2]].clone()], [v0, v0.clone(), v0[:held[2]].clone()]
    for s in (1, 0, 2):
        f.pool.alloc(s, held[s], 3)
        k, v = _kv(torch, g, 3, 3, hd, torch.float32)
        rows.write(list(range(held[s], held[s] + 3)), [s] * 3)
        ops.kv_store(k, v, f.pool, 0, 3, rows)
        f.k[s] = torch.cat([f.k[s], q8_util.stored(k)])
        f.v[s] = torch.cat([f.v[s], q8_util.stored(v)])
    for s in range(3):
        m = len(f.k[s])
        r = RowMeta(m)
        r.write(list(range(m)), [s] * m)
        k, v = _load(torch, f.pool, r, m, torch.float32)
        assert _same(k.double(), f.k[s]) and _same(v.double(), f.v[s]), s
    chunks = [(s, [len(f.k[s]) - 1]) for s in range(3)]
    q = f.query(3, 9, torch.float32)
    y = torch.zeros_like(q)
    ops.attn(q, f.pool, 0, y, _spec(chunks, 9, hd))
    want, bound = f.want(q, chunks, 0, 0.0)
    q8_util.check("forks", y, want, bound, y.dtype)
    # rollback: the last tokens go, new ones take their place
    f.pool.truncate(1, n - 2)
    f.pool.alloc(1, n - 2, 4)
    k, v = _kv(torch, g, 4, 3, hd, torch.float32)
    rows.write(list(range(n - 2, n + 2)), [1] * 4)
    ops.kv_store(k, v, f.pool, 0, 4, rows)
    f.k[1] = torch.cat([f.k[1][:n - 2], q8_util.stored(k)])
    r = RowMeta(n + 2)
    r.write(list(range(n + 2)), [1] * (n + 2))
    lk, _ = _load(torch, f.pool, r, n + 2, torch.float32)
    assert _same(lk.double(), f.k[1])


@pytest.mark.parametrize("tokens", [1, 3, 4, 5, 15, 16, 18, 32])
def test_block_copy(torch_cuda, tokens):
    """Slots [0, tokens) move, the others of the destination stay."""
    torch = torch_cuda
    pool = KvPool(ArenaSpec([64, 64], 4), 2, 72, layers=1, page_len=32, kv_dtype="e4m3")
    pool.alloc(0, 0, 64)
    pool.alloc(1, 0, 64)
    g = torch.Generator(device="cuda").manual_seed(2)
    k, v = _kv(torch, g, 128, 2, 72, torch.float32)
    rows = RowMeta(128)
    rows.write(list(range(64)) * 2, [0] * 64 + [1] * 64)
    ops.kv_store(k, v, pool, 0, 128, rows)
    ks, vs = q8_util.stored(k), q8_util.stored(v)
    src, dst = pool.arena.table_of(0)[1], pool.arena.table_of(1)[0]
    ops.block_copy(pool, [(src, dst, tokens)])
    ks[64:64 + tokens], vs[64:64 + tokens] = ks[32:32 + tokens].clone(), vs[32:32 + tokens].clone()
    lk, lv = _load(torch, pool, rows, 128, torch.float32)
    assert _same(lk.double(), ks) and _same(lv.double(), vs)


# ------------------------------------------------------------ whole steps


@pytest.mark.parametrize("src", ["f32", "f16"])
@pytest.mark.parametrize("nq,nkv,hd,rot,norm", [(32, 8, 128, 128, True), (14, 2, 64, 64, False), (8, 4, 96, 48, True),
                                                (4, 2, 256, 64, False)])
def test_rotary_step(torch_cuda, src, nq, nkv, hd, rot, norm):
    """attn_step with rope, norms, a query stride and a gate equals the separate
    calls: rope_rows on q and k, kv_store, attn, gate."""
    torch = torch_cuda
    dt = _dt(torch, src)
    lens, new = [300, 17, 90], [1, 17, 3]
    f = Filled(torch, [n - c for n, c in zip(lens, new)], nkv, hd, seed=hd, budget=lens)
    chunks = [(s, list(range(n - c, n))) for s, (n, c) in enumerate(zip(lens, new))]
    for s, (n, c) in enumerate(zip(lens, new)):
        f.pool.alloc(s, n - c, c)
    m = sum(new)
    spec = _spec(chunks, nq, hd)
    ang = torch.arange(400, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))
    w = [1 + 0.1 * torch.randn(hd, device="cuda", generator=f.g) for _ in range(2)] if norm else [None, None]
    rope = Rope(ang.cos().float().numpy(), ang.sin().float().numpy(), rot, q_norm=w[0], k_norm=w[1], eps=1e-5)
    qg = torch.randn(m, nq, 2 * hd, device="cuda", generator=f.g).to(dt)
    k, v = _kv(torch, f.g, m, nkv, hd, dt)
    y = torch.zeros(m, nq, hd, device="cuda")
    ops.attn_step(f.pool, 0, spec, qg[..., :hd], y, q_stride=2 * hd, gate=qg[..., hd:], gate_stride=2 * hd, k_src=k,
                  v_src=v, rope=rope)
    got = _load(torch, f.pool, spec.args, m, torch.float32)
    kr = k.clone()
    rope_rows(kr, nkv, rope, spec.args, m, norm_w=w[1])
    assert _same(got[0].double(), q8_util.stored(kr)) and _same(got[1].double(), q8_util.stored(v))
    qr = qg[..., :hd].float().contiguous()
    rope_rows(qr, nq, rope, spec.args, m, norm_w=w[0])
    at = 0
    for s, c in enumerate(new):
        f.k[s] = torch.cat([f.k[s], q8_util.stored(kr[at:at + c])])
        f.v[s] = torch.cat([f.v[s], q8_util.stored(v[at:at + c])])
        at += c
    want, bound = f.want(qr, chunks, 0, 0.0)
    sig = 1 / (1 + torch.exp(-qg[..., hd:].double()))
    # (the rotated query's own roundings, 2^-22 of it, are within the bound's two of an f32 query's)
    q8_util.check(f"step {nq}/{nkv}x{hd} {src}", y, want * sig, bound * sig + want.abs() * 2.0 ** -20, y.dtype)


def test_append_and_attention_in_one_call(torch_cuda):
    """kv_store_attn equals kv_store and attn, bit for bit, in outputs and pool."""
    torch = torch_cuda
    for lens, new, nq, nkv, hd in (([600, 31, 1, 64], [1, 1, 1, 1], 32, 8, 128), ([300, 20], [4, 4], 8, 4, 256),
                                   ([64, 500], [64, 1], 14, 2, 64)):
        out = []
        for fused in (True, False):
            f = Filled(torch, [n - c for n, c in zip(lens, new)], nkv, hd, seed=1, budget=lens)
            for s, (n, c) in enumerate(zip(lens, new)):
                f.pool.alloc(s, n - c, c)
            m = sum(new)
            spec = _spec([(s, list(range(n - c, n))) for s, (n, c) in enumerate(zip(lens, new))], nq, hd)
            q = f.query(m, nq, torch.float16)
            k, v = _kv(torch, f.g, m, nkv, hd, torch.float16)
            y = torch.zeros(m, nq, hd, device="cuda")
            if fused:
                ops.kv_store_attn(k, v, q, f.pool, 0, y, spec)
            else:
                ops.kv_store(k, v, f.pool, 0, m, spec.args)
                ops.attn(q, f.pool, 0, y, spec)
            lk, lv = _load(torch, f.pool, spec.args, m, torch.float32)
            assert _same(lk.double(), q8_util.stored(k)) and _same(lv.double(), q8_util.stored(v))
            out.append((y, lk, lv))
        assert all(torch.equal(a, b) for a, b in zip(*out))


def test_captured_step(torch_cuda):
    """Page allocation, append, plan, attention and read-back of a decode step
    captured once and replayed while positions move, with eager work between."""
    torch = torch_cuda
    nq, nkv, hd, b = 8, 2, 128, 3
    lens = [30, 100, 13]
    f = Filled(torch, lens, nkv, hd, budget=[n + 40 for n in lens], extra=2)
    rows = RowMeta(b)
    plan = ops.DevicePlan(f.pool, max_m=b, q_heads=nq)
    q = torch.zeros(b, nq, hd, device="cuda", dtype=torch.float16)
    k, v = (torch.zeros(b, nkv, hd, device="cuda", dtype=torch.float16) for _ in range(2))
    y = torch.zeros(b, nq, hd, device="cuda")
    lk, lv = (torch.zeros(b, nkv, hd, device="cuda") for _ in range(2))
    spec = ops.AttnSpec(q_heads=nq, window=0, scale=1 / math.sqrt(hd), m=b, causal=True, seq=None, args=rows)

    def body():
        f.pool.alloc_rows(rows, b)
        ops.kv_store(k, v, f.pool, 0, b, rows)
        plan.build(spec, q, y)
        plan.attn(0, q, y)
        ops.kv_load(lk, lv, f.pool, 0, b, rows)

    def inputs(step):
        rows.write([n + step for n in lens], list(range(b)))
        q.copy_(f.query(b, nq, torch.float16))
        nk, nv = _kv(torch, f.g, b, nkv, hd, torch.float16)
        k.copy_(nk)
        v.copy_(nv)
        for s in range(b):
            f.k[s] = torch.cat([f.k[s], q8_util.stored(nk[s:s + 1])])
            f.v[s] = torch.cat([f.v[s], q8_util.stored(nv[s:s + 1])])

    def verify(step):
        torch.cuda.synchronize()
        f.pool.status()
        chunks = [(s, [n + step]) for s, n in enumerate(lens)]
        want, bound = f.want(q, chunks, 0, 0.0)
        q8_util.check(f"captured step {step}", y, want, bound, y.dtype)
        for s in range(b):
            assert _same(lk[s].double(), f.k[s][-1]) and _same(lv[s].double(), f.v[s][-1])

    inputs(0)
    body()
    verify(0)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            body()
    torch.cuda.current_stream().wait_stream(side)
    for step in range(1, 22):
        inputs(step)
        y.fill_(5.0)
        graph.replay()
        verify(step)
        torch.randn(1000, device="cuda").sum()  # eager work between replays


def test_many_layers_and_head_dims(torch_cuda):
    """Layers of different head_dims keep to their own planes."""
    torch = torch_cuda
    hds = [64, 200, 128]
    pool = make_pool([50], 2, 64, kv_dtype="e4m3", layers=3, head_dims=hds)
    pool.alloc(0, 0, 50)
    rows = RowMeta(50)
    rows.write(list(range(50)), [0] * 50)
    g = torch.Generator(device="cuda").manual_seed(6)
    kv = [_kv(torch, g, 50, 2, hd, torch.float32) for hd in hds]
    for layer, (k, v) in enumerate(kv):
        ops.kv_store(k, v, pool, layer, 50, rows)
    for layer, (k, v) in enumerate(kv):
        lk, lv = _load(torch, pool, rows, 50, torch.float32, layer)
        assert _same(lk.double(), q8_util.stored(k)) and _same(lv.double(), q8_util.stored(v))


# ------------------------------------------------------------------ refusals


def _refused(text, fn):
    with pytest.raises(ThubanError) as e:
        fn()
    assert text in str(e.value), str(e.value)


def test_refusals(torch_cuda):
    torch = torch_cuda
    f = Filled(torch, [20, 20], 2, 64)
    rows = RowMeta(4)
    x = torch.zeros(4, 2, 64, device="cuda")
    w = torch.zeros(2, 4, 64, dtype=torch.int16, device="cuda")
    rows.write([3, 4, 3], [0, 0, 0])
    _refused("two rows append position 3 of sequence 0", lambda: ops.kv_store(x, x, f.pool, 0, 3, rows))
    rows.write([3, 3, 4], [0, 1, 0])
    ops.kv_store(x, x, f.pool, 0, 3, rows)  # one position of two sequences
    spec = ops.AttnSpec(q_heads=2, window=0, scale=1.0, m=2, causal=True, seq=None, args=rows)
    rows.write([3, 3], [1, 1])
    _refused("two rows append", lambda: ops.kv_store_attn(x, x, x, f.pool, 0, x.clone(), spec))
    rows.write([40], [0])
    _refused("pages must cover", lambda: ops.kv_load(x, x.clone(), f.pool, 0, 1, rows))
    _refused("pages must cover", lambda: ops.kv_store(x, x, f.pool, 0, 1, rows))
    rows.write([0], [2])
    _refused("out of range", lambda: ops.kv_load(x, x.clone(), f.pool, 0, 1, rows))
    rows.write([0], [0])
    _refused("row meta holds 1 rows", lambda: ops.kv_load(x, x.clone(), f.pool, 0, 2, rows))
    _refused("layer 1 out of range", lambda: ops.kv_load(x, x.clone(), f.pool, 1, 1, rows))
    _refused("16-byte aligned",
             lambda: ops.kv_load(x.data_ptr() + 4, x.data_ptr(), f.pool, 0, 1, rows))
    _refused("dtypes differ", lambda: ops.kv_load(x, x.half(), f.pool, 0, 1, rows))
    ops.kv_load(x, x.clone(), f.pool, 0, 0, rows)
    _refused("gather and scatter move 16-bit words", lambda: ops.kv_gather(f.pool, 0, 0, 0, 4, w, w))
    _refused("gather and scatter move 16-bit words", lambda: ops.kv_scatter(f.pool, 0, 0, 0, 4, w, w))
    _refused("gather and scatter move 16-bit words", lambda: ops.kv_gather_batch(f.pool, [(0, 0, 0, 4)], w, w))
    _refused("8-bit pool has no 16-bit words", lambda: f.pool.read_layer(0))
    _refused("take no flags", lambda: ops.DevicePlan(f.pool, 4, 2, append=True))
    _refused("take no flags", lambda: ops.DevicePlan(f.pool, 4, 2, prefill=True))
    p16 = make_pool([20], 2, 64, kv_dtype="f16")
    p16.alloc(0, 0, 20)
    _refused("thb_kv_load reads 8-bit pools", lambda: ops.kv_load(x, x.clone(), p16, 0, 1, rows))
