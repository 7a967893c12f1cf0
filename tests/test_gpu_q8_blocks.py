"""Chunks over 8-bit pages large enough for prefill blocks (8 query groups, one
workgroup per CU: many KV heads and short partitions here), and appends large enough for four
rows a lane, against 64 bits."""

import ctypes
import math
import random

import pytest

from flint_amd import _lib, ops
from flint_amd.pool import RowMeta
from flint_amd.rope import Rope, kv_store_rope, rope_rows
from tests import q8_util
from tests.gpu_util import make_pool, scattered_alloc
from tests.test_gpu_q8 import Filled, _dt, _kv, _load, _same, _spec

pytestmark = pytest.mark.gpu


def _want(f, q, chunks, window, cap, yd):
    """y and bound; a 16-bit output's probabilities are rounded to f16 (each off
    by at most 2^-11 of itself): 2^-11 of the weighted magnitudes more."""
    want, bound = f.want(q, chunks, window, cap)
    if yd != "f32":
        v = f.v
        f.v = [x.abs() for x in v]
        mag, _ = f.want(q, chunks, window, cap)
        f.v = v
        bound = bound + mag.nan_to_num() * 2.0 ** -11
    return want, bound


BLOCKS = [
    # nq, nkv, hd, page, [(tokens, new)], q, y, window, softcap, part_len
    (64, 32, 128, 16, [(300, 100)], "f16", "f16", 0, 0.0, 128),
    (64, 32, 128, 16, [(300, 100)], "f16", "f32", 0, 0.0, 128),
    (32, 32, 64, 16, [(300, 100)], "f32", "f32", 0, 0.0, 64),
    (32, 32, 96, 16, [(300, 100)], "f32", "f16", 0, 0.0, 64),
    (64, 16, 128, 32, [(700, 160), (70, 70), (333, 120), (9, 1)], "bf16", "bf16", 100, 0.0, 64),
    (32, 16, 128, 16, [(400, 150)], "f32", "f32", 0, 30.0, 64),
    (32, 16, 80, 64, [(401, 150)], "f16", "f16", 37, 30.0, 64),
    (48, 16, 64, 16, [(350, 33)] * 6, "f16", "f32", 0, 20.0, 128),
    (32, 32, 64, 16, [(300, 140)], "f32", "f32", 0, 0.0, 64),
    (32, 32, 96, 16, [(300, 140)], "f32", "f16", 0, 0.0, 64),
    (48, 16, 64, 16, [(350, 60), (40, 5), (90, 90), (200, 50), (90, 60), (333, 60)], "f16", "f32", 0, 20.0, 128),
    # two query groups a wave: eight times the workgroups
    (256, 64, 128, 16, [(260, 64)], "f16", "f16", 0, 0.0, 32),
    (256, 64, 128, 16, [(260, 64)], "bf16", "f32", 0, 25.0, 32),
    (256, 64, 112, 16, [(259, 63)], "f16", "f32", 200, 0.0, 32),
]


@pytest.mark.parametrize("nq,nkv,hd,page,seqs,qd,yd,window,cap,part", BLOCKS)
def test_blocks(torch_cuda, nq, nkv, hd, page, seqs, qd, yd, window, cap, part):
    torch = torch_cuda
    f = Filled(torch, [n for n, _ in seqs], nkv, hd, page, seed=hd, part_len=part, src="bf16")
    chunks = [(s, list(range(n - new, n))) for s, (n, new) in enumerate(seqs)]
    spec = _spec(chunks, nq, hd, window, cap)
    q = f.query(spec.m, nq, _dt(torch, qd))
    y = torch.full((spec.m, nq, hd), 3.0, dtype=_dt(torch, yd), device="cuda")
    ops.attn(q, f.pool, 0, y, spec)
    want, bound = _want(f, q, chunks, window, cap, yd)
    q8_util.check(f"blocks {nq}/{nkv}x{hd}", y, want, bound, y.dtype)
    again = torch.zeros_like(y)
    ops.attn(q, f.pool, 0, again, spec)
    assert torch.equal(y, again)
    if nq > 64:
        return
    # the no-allocation call has no scratch for expanded keys: decode items (nor for
    # the partial results of 256 heads)
    y2 = torch.zeros_like(y)
    c = ops._spec_c(spec, q, y2)
    _lib.check(_lib.lib().thb_attn_noalloc(f.pool.handle, 0, q.data_ptr(), y2.data_ptr(), ctypes.byref(c),
                                           spec.args.handle, torch.cuda.current_stream().cuda_stream))
    want, bound = f.want(q, chunks, window, cap)
    q8_util.check(f"no-allocation {nq}/{nkv}x{hd}", y2, want, bound, y.dtype)


@pytest.mark.parametrize("qd,yd", [("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("hd", [64, 128])
def test_scales_from_step_to_step(torch_cuda, hd, qd, yd):
    """Scales of V that rise and fall by 2^60 from one run of 32 keys to the next,
    zero keys and values among them."""
    torch = torch_cuda
    n, new, nkv, nq = 384, 150, 32, 32
    f = Filled(torch, [n], nkv, hd, part_len=128)
    g = f.g
    k, v = _kv(torch, g, n, nkv, hd, torch.float32)
    e = torch.tensor([0, -30, 30, 5, -25, -60, 40, -1, 20, 19, 50, -50], device="cuda").repeat_interleave(32)
    v = v * torch.exp2(e.float())[:, None, None]
    v[40:50] = 0
    k[200:290] = 0
    v[64:96] = 0
    rows = RowMeta(n)
    rows.write(list(range(n)), [0] * n)
    ops.kv_store(k, v, f.pool, 0, n, rows)
    f.k[0], f.v[0] = q8_util.stored(k), q8_util.stored(v)
    chunks = [(0, list(range(n - new, n)))]
    spec = _spec(chunks, nq, hd)
    q = f.query(new, nq, _dt(torch, qd))
    y = torch.zeros(new, nq, hd, dtype=torch.float32, device="cuda") if yd == "f32" else \
        torch.zeros(new, nq, hd, dtype=torch.bfloat16, device="cuda")  # (f16 has no room for these values)
    ops.attn(q, f.pool, 0, y, spec)
    want, bound = _want(f, q, chunks, 0, 0.0, yd)
    q8_util.check(f"scales by step x{hd}", y, want, bound, y.dtype)


@pytest.mark.parametrize("hd,new", [(64, 100), (128, 70), (128, 100)])
def test_nan_in_blocks(torch_cuda, hd, new):
    """A NaN token reaches the rows of its chunk that read it and no other."""
    torch = torch_cuda
    n, nkv, nq = 200, 64, 128
    f = Filled(torch, [n], nkv, hd, part_len=64, budget=[n + 64])
    pos = list(range(n - new, n))
    bad = n - new + new // 2
    rows = RowMeta(8)
    rows.write([bad], [0])
    x = torch.full((1, nkv, hd), math.inf, device="cuda")
    z = torch.ones(1, nkv, hd, device="cuda")
    for k, v in ((x, z), (z, x)):
        ops.kv_store(k, v, f.pool, 0, 1, rows)
        f.k[0][bad], f.v[0][bad] = q8_util.stored(k)[0], q8_util.stored(v)[0]
        spec = _spec([(0, pos)], nq, hd)
        q = f.query(new, nq, torch.float16)
        y = torch.zeros(new, nq, hd, device="cuda")
        ops.attn(q, f.pool, 0, y, spec)
        first = pos.index(bad)
        assert y[first:].isnan().all() and not y[:first].isnan().any()
        want, bound = f.want(q[:first], [(0, pos[:first])], 0, 0.0)
        q8_util.check("rows before the NaN", y[:first], want, bound, y.dtype)


def test_slots_behind_the_chunk(torch_cuda):
    """What the slots behind the last key hold (a longer sequence's huge and NaN
    vectors, on pages since reused) does not touch a chunk's precision."""
    torch = torch_cuda
    n, new, nkv, hd = 203, 150, 32, 128
    pool = make_pool([n + 53], nkv, hd, page_len=16, kv_dtype="e4m3", part_len=64)
    pool.alloc(0, 0, n + 53)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = _kv(torch, g, n + 53, nkv, hd, torch.float32)
    k[n:] *= 2.0 ** 40
    v[n:] *= 2.0 ** 60
    k[n + 2], v[n + 3] = math.nan, math.inf
    rows = RowMeta(512)
    rows.write(list(range(n + 53)), [0] * (n + 53))
    ops.kv_store(k, v, pool, 0, n + 53, rows)
    pool.truncate(0, n)
    pos = list(range(n - new, n))
    spec = _spec([(0, pos)], nkv, hd)
    q = torch.randn(new, nkv, hd, device="cuda", generator=g)
    y = torch.zeros_like(q)
    ops.attn(q, pool, 0, y, spec)
    want, bound = q8_util.attend(q, q8_util.stored(k[:n]), q8_util.stored(v[:n]), q8_util.row_ranges(pos, 0),
                                 1 / math.sqrt(hd))
    q8_util.check("slots behind the chunk", y, want, bound, y.dtype)


# ------------------------------------------------------- appends, four rows a lane


def _token_order(rng, m, budget):
    """m different positions below budget: runs, single tokens, falling runs."""
    free, out, p = budget, [], rng.randrange(4)
    while len(out) < m:
        run = rng.choice([1, 1, 2, 3, 4, 5, 8, 33, 70])
        run = min(run, m - len(out))
        r = list(range(p, p + run))
        out += r[::-1] if rng.random() < 0.2 else r
        p += run + rng.choice([0, 0, 0, 1, 2, 3])
    assert p <= free + 3 * m and max(out) < budget
    return out


@pytest.mark.parametrize("nkv,hd,page,m", [(16, 512, 16, 301), (96, 72, 32, 201), (128, 64, 16, 300), (40, 200, 64, 300),
                                           (64, 128, 256, 262)])
@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
def test_rows_in_any_order(torch_cuda, nkv, hd, page, m, src):
    torch = torch_cuda
    rng = random.Random(hd)
    budget = 4 * m
    lens = [budget, budget]
    pool = make_pool(lens, nkv, hd, page_len=page, kv_dtype="e4m3", extra_pages=2)
    scattered_alloc(pool, lens, rng, page)
    half = m // 2 + 1
    pos = _token_order(rng, half, budget) + _token_order(rng, m - half, budget)
    own = [0] * half + [1] * (m - half)
    g = torch.Generator(device="cuda").manual_seed(m)
    k, v = _kv(torch, g, m, nkv, hd, _dt(torch, src))
    k[7], v[9], v[10] = math.inf, math.nan, 0.0
    # everything holds other values first: rows not appended keep them
    old = RowMeta(budget)
    ok, ov = _kv(torch, g, budget, nkv, hd, torch.float32)
    for s in range(2):
        old.write(list(range(budget)), [s] * budget)
        ops.kv_store(ok, ov, pool, 0, budget, old)
    rows = RowMeta(m)
    rows.write(pos, own)
    ops.kv_store(k, v, pool, 0, m, rows)
    f32 = torch.float32
    lk, lv = _load(torch, pool, rows, m, f32)
    assert _same(q8_util.stored(k).to(f32), lk) and _same(q8_util.stored(v).to(f32), lv)
    for s in range(2):
        old.write(list(range(budget)), [s] * budget)
        ak, av = _load(torch, pool, old, budget, f32)
        wk, wv = q8_util.stored(ok).to(f32), q8_util.stored(ov).to(f32)
        at = torch.tensor([p for p, o in zip(pos, own) if o == s], device="cuda")
        sel = torch.tensor([i for i, o in enumerate(own) if o == s], device="cuda")
        wk[at], wv[at] = q8_util.stored(k).to(f32)[sel], q8_util.stored(v).to(f32)[sel]
        assert _same(ak, wk) and _same(av, wv)


@pytest.mark.parametrize("src", ["f32", "f16"])
@pytest.mark.parametrize("nkv,hd,rot,norm", [(64, 128, 64, True), (72, 96, 96, False)])
def test_rotary_append_of_a_chunk(torch_cuda, src, nkv, hd, rot, norm):
    torch = torch_cuda
    m = 270
    dt = _dt(torch, src)
    pool = make_pool([m + 9], nkv, hd, page_len=16, kv_dtype="e4m3")
    pool.alloc(0, 0, m + 9)
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = _kv(torch, g, m, nkv, hd, dt)
    rows = RowMeta(m)
    rows.write(list(range(9, m + 9)), [0] * m)
    ang = torch.arange(400, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))
    w = 1 + 0.1 * torch.randn(hd, device="cuda", generator=g) if norm else None
    rope = Rope(ang.cos().float().numpy(), ang.sin().float().numpy(), rot, q_norm=w, k_norm=w, eps=1e-5)
    kv_store_rope(k, v, pool, 0, m, rows, rope)
    kr = k.clone()
    rope_rows(kr, nkv, rope, rows, m, norm_w=w)
    lk, lv = _load(torch, pool, rows, m, torch.float32)
    assert _same(q8_util.stored(kr).float(), lk) and _same(q8_util.stored(v).float(), lv)
