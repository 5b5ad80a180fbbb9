"""Decoding operators (fudanocr_amd/decode.py): refusals on the CPU, the kernels against plain 64-bit forms on the GPU.

Tolerances.  With u = 2^-24 (fp32 arithmetic) and u_t = eps(type) / 2: a score c q.k is off by at most
d = (dim + 4) u c sum|q||k| plus 2^-21 |c q.k| for the exponent's argument, so a weight by a factor e^{+-d}, a normalised weight by
2 d (numerator and denominator), plus the sums' own (keys + 4) u; 16-bit types round each weight once more (u_t) before the
product with v.  An output is off by at most (2 d + (keys + 8) u + [16 bit] 2 u_t) sum p|v| / sum p, plus the final rounding
u_t |o|."""
import math
import os
import random
import subprocess

import pytest
import torch

from fudanocr_amd import decode as D

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


# ------------------------------------------------------------------------------------------------ building blocks
class Pool:
    """a paged cache with `lens` tokens per sequence, pages scattered, unused slots and pages holding NaN; CPU copies of the
    dense keys / values in 64 bits"""

    def __init__(self, lens, kv_heads, dim, page, dtype, seed=0, extra=2, table_ld=None, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lens]
        ld = table_ld or max(1, max(need))
        total = sum(need) + extra
        perm = torch.randperm(total, generator=g).tolist()
        self.k = torch.full((total, kv_heads, page, dim), float("nan"))
        self.v = self.k.clone()
        self.table = torch.full((len(lens), ld), -7, dtype=torch.int32)
        self.dense = []
        at = 0
        for s, n in enumerate(lens):
            self.table[s, :need[s]] = torch.tensor(perm[at:at + need[s]], dtype=torch.int32)
            at += need[s]
            kv = torch.randn(2, n, kv_heads, dim, generator=g).to(dtype)
            self.dense.append(kv.double())
            for j in range(need[s]):
                rows = slice(j * page, min(n, (j + 1) * page))
                m = rows.stop - rows.start
                pg = int(self.table[s, j])
                self.k[pg, :, :m] = kv[0, rows].float().transpose(0, 1)
                self.v[pg, :, :m] = kv[1, rows].float().transpose(0, 1)
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.k, self.v = self.k.to(dtype).to(device), self.v.to(dtype).to(device)
        self.dev_table, self.dev_lens = self.table.to(device), self.lens.to(device)

    @property
    def args(self):
        return self.k, self.v, self.dev_table, self.dev_lens


def reference(q, dense, starts, news, causal, scale):
    """64-bit output and its tolerance per element (module docstring); rows of no sequence are NaN in both"""
    tokens, heads, dim = q.shape
    out = torch.full((tokens, heads, dim), float("nan"), dtype=torch.float64)
    tol = torch.full_like(out, float("nan"))
    u, ut = 2.0 ** -24, torch.finfo(q.dtype).eps / 2
    for (k, v), t0, n in zip(dense, starts, news):
        length, kvh = k.shape[0], k.shape[1]
        grp = heads // kvh
        for i in range(n):
            vis = max(0, length - n + 1 + i) if causal else length
            if vis == 0:
                out[t0 + i], tol[t0 + i] = 0.0, 0.0
                continue
            qi = q[t0 + i].double().view(kvh, grp, dim)
            kk, vv = k[:vis].permute(1, 2, 0), v[:vis].transpose(0, 1)
            s = qi @ kk * scale
            mag = (qi.abs() @ kk.abs() * scale).amax(-1, keepdim=True)
            p = torch.softmax(s, -1)
            o = p @ vv
            d = (dim + 4) * u * mag + 2.0 ** -21 * s.abs().amax(-1, keepdim=True)
            rel = 2 * d + (vis + 8) * u + (2 * ut if q.dtype != torch.float32 else 0.0)
            out[t0 + i] = o.view(heads, dim)
            tol[t0 + i] = (rel * (p @ vv.abs()) + ut * o.abs() + 1e-30).view(heads, dim)
    return out, tol


def check(got, ref, tol, keep=None):
    got = got.double().cpu()
    owned = ~torch.isnan(ref)
    err = (got - ref).abs()
    bad = owned & ~(err <= tol)
    assert not bad.any(), "%d of %d off, worst %g x its tolerance" % (
        int(bad.sum()), int(owned.sum()), float((err / tol.clamp_min(1e-30))[bad].max()))
    if keep is not None:
        assert torch.equal(got[~owned], keep.double().cpu()[~owned])


def starts_of(news, first=0):
    s = [first]
    for n in news:
        s.append(s[-1] + n)
    return s


# ----------------------------------------------------------------------------------------------------- CPU: refusals
def test_index_arithmetic_on_the_cpu(tmp_path):
    """csrc/paged_index.h compiled for the host with sanitizers, over whole ranges of lengths, tables and offsets, bad ones
    among them (tests/cpp/paged_index_check.cpp)"""
    exe = str(tmp_path / "paged_index_check")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-I",
                           os.path.join(ROOT, "fudanocr_amd", "csrc"), os.path.join(ROOT, "tests", "cpp", "paged_index_check.cpp"),
                           "-o", exe])
    out = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout[-2000:] + out.stderr[-2000:]


def _cpu_cache(page=16, dim=64, heads=2, seqs=3, ld=2, dtype=torch.float32):
    k = torch.zeros(8, heads, page, dim, dtype=dtype)
    return [k, k.clone(), torch.zeros(seqs, ld, dtype=torch.int32), torch.zeros(seqs, dtype=torch.int32)]


def _raises(match, f, *a, **kw):
    with pytest.raises(RuntimeError, match=match):
        f(*a, **kw)


def test_attention_refuses_bad_arguments():
    c, q = _cpu_cache(), torch.zeros(3, 4, 64)
    _raises("on the GPU", D.paged_attention, q, *c)
    _raises("on the GPU", D.paged_append, q[:, :2], q[:, :2], *c)
    _raises("power of two", D.paged_attention, q, *_cpu_cache(page=12))
    _raises("power of two", D.paged_attention, q, *_cpu_cache(page=4))
    _raises("head dim", D.paged_attention, torch.zeros(3, 4, 96), *_cpu_cache(dim=96))
    _raises("of one type", D.paged_attention, q, c[0], c[1].half(), *c[2:])
    _raises("of one type", D.paged_attention, q.double(), c[0].double(), c[1].double(), *c[2:])
    _raises("contiguous and on one device", D.paged_attention, q, c[0].transpose(1, 2).contiguous().transpose(1, 2), *c[1:])
    _raises("table must be", D.paged_attention, q, c[0], c[1], c[2].long(), c[3])
    _raises("kv_lens must be", D.paged_attention, q, c[0], c[1], c[2], c[3][:2])
    _raises("q_start must be", D.paged_attention, q, *c, q_start=torch.zeros(3, dtype=torch.int32))
    _raises("q must be", D.paged_attention, q.half(), *c)
    _raises("q must be", D.paged_attention, torch.zeros(3, 4, 128), *c)
    _raises("contiguous rows", D.paged_attention, torch.zeros(3, 64, 4).transpose(1, 2), *c)
    _raises("3 heads over a cache of 2", D.paged_attention, torch.zeros(3, 3, 64), *c)
    _raises("same number of rows", D.paged_attention, torch.zeros(4, 4, 64), *c)
    for scale in (0.0, -1.0, math.inf, math.nan):
        _raises("scale", D.paged_attention, q, *c, scale=scale)
    _raises("out must have q's shape", D.paged_attention, q, *c, out=torch.zeros(4, 4, 64))
    _raises("rows of its own", D.paged_attention, q, *c, out=torch.zeros(1, 4, 64).expand(3, 4, 64))
    _raises("wants a gradient", D.paged_attention, q.clone().requires_grad_(True), *c)
    _raises("wants a gradient", D.paged_append, torch.zeros(3, 2, 64, requires_grad=True), torch.zeros(3, 2, 64), *c)
    with torch.no_grad():
        _raises("on the GPU", D.paged_attention, q.clone().requires_grad_(True), *c)
    _raises("share q's memory", D.paged_attention, q, *c, out=q)
    _raises("k_new must be", D.paged_append, q, q, *c)
    _raises("same tokens", D.paged_append, torch.zeros(3, 2, 64), torch.zeros(6, 2, 64), *c)


def test_beam_operators_refuse_bad_arguments():
    x, s = torch.zeros(2, 3, 7), torch.zeros(2, 3)
    _raises("on the GPU", D.beam_select, x, s)
    _raises("logits must be", D.beam_select, x.double(), s)
    _raises("logits must be", D.beam_select, x[0], s)
    _raises("wants a gradient", D.beam_select, x.clone().requires_grad_(True), s)
    _raises("1 to 64", D.beam_select, torch.zeros(1, 65, 7), torch.zeros(1, 65))
    _raises("n at most", D.beam_select, torch.zeros(1, 2, 3), torch.zeros(1, 2), n=7)
    _raises("contiguous rows", D.beam_select, torch.zeros(2, 7, 3).transpose(1, 2), s)
    _raises("scores must be", D.beam_select, x, s.double())
    _raises("need an eos", D.beam_select, x, s, torch.zeros(2, 3, dtype=torch.bool))
    _raises("finished must be", D.beam_select, x, s, torch.zeros(2, 3), eos=1)
    _raises("inside the vocabulary", D.beam_select, x, s, eos=7)
    p, t, sp = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(6, 2, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)
    pages = [torch.zeros(8, 2, 16, 64)]
    _raises("on the GPU", D.beam_reorder, p, t, sp, sp, pages)
    _raises("table must be", D.beam_reorder, p, t[:5], sp, sp, pages)
    _raises("parents must be", D.beam_reorder, p.long(), t, sp, sp, pages)
    _raises("spare must be", D.beam_reorder, p, t, sp, sp[:4], pages)
    _raises("no page tensors", D.beam_reorder, p, t, sp, sp, [])
    _raises("of one", D.beam_reorder, p, t, sp, sp, pages + [torch.zeros(8, 2, 16, 64).half()])
    _raises("power of two", D.beam_reorder, p, t, sp, sp, [torch.zeros(8, 2, 12, 64)])
    _raises("16-byte units", D.beam_reorder, p, t, sp, sp, [torch.zeros(8, 2, 16, 3)])
    _raises("table_out must be", D.beam_reorder, p, t, sp, sp, pages, t[:, :1])
    _raises("in a cache of 20", D.PagedCache(2, 20, 2, 64, device="cpu").advance, 21)


def test_c_entries_refuse_before_they_launch():
    """the C ABI's own checks: an error code and a message, nothing launched (there is no GPU to launch on)"""
    from fudanocr_amd import _lib
    lib = _lib.load()
    p = 4096                                                   # a pointer that is never followed
    ok = dict(q=p, ldt=256, ldh=64, k=p, v=p, table=p, lens=p, qs=None, o=p, ldto=256, ldho=64, ws=None, wsb=0, tokens=3, seqs=3,
              heads=4, kvh=2, dim=64, page=16, ld=2, pages=8, max_q=1, max_kv=32, scale=0.1, causal=1, dt=0)

    def call(**kw):
        a = {**ok, **kw}
        return lib.focr_paged_attention_fwd(*a.values(), None), lib.focr_last_error().decode()
    for kw, text in ((dict(dt=3), "dtype"), (dict(dim=65), "head dim"), (dict(page=24), "power of two"), (dict(page=2048), "power of two"),
                     (dict(k=p + 8), "aligned"), (dict(o=None), "null"), (dict(heads=3), "multiple"), (dict(pages=0), "empty"),
                     (dict(ws=p + 4), "aligned"), (dict(max_kv=2 ** 31 - 1), "max_kv"), (dict(tokens=4), "tokens / seqs"), (dict(tokens=6), "max_q"), (dict(scale=0.0), "scale"), (dict(tokens=-1), "range")):
        rc, msg = call(**kw)
        assert rc == -1 and text in msg, (kw, rc, msg)
    assert call(tokens=0)[0] == 0 and call(seqs=0)[0] == 0


# ---------------------------------------------------------------------------------------------------- GPU: attention
MIXES = [
    ("single", [1, 1, 1, 1], [1, 16, 17, 200]),                       # one token each: alone, page borders, several tiles
    ("ragged", [1, 0, 3, 40, 1, 130, 17], [1, 5, 3, 70, 300, 130, 400]),
    ("late", [5, 2, 33], [3, 0, 20]),                                 # more new tokens than the cache holds: empty rows
    ("chunk", [257], [700]),
]


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (6, 2), (8, 1)])
@pytest.mark.parametrize("mix", MIXES, ids=[m[0] for m in MIXES])
def test_attention_against_64_bits(dtype, dim, heads, kv_heads, mix):
    _, news, lens = mix
    pool = Pool(lens, kv_heads, dim, 16, dtype, seed=dim + heads)
    g = torch.Generator().manual_seed(5)
    first, tail = 2, 3                                                # rows of no sequence on both sides
    starts = starts_of(news, first)
    q = (2 * torch.randn(starts[-1] + tail, heads, dim, generator=g)).to(dtype)
    scale = dim ** -0.5
    keep = torch.randn(q.shape, generator=g).to(dtype).cuda()
    for causal in (True, False):
        ref, tol = reference(q, pool.dense, starts, news, causal, scale)
        out = keep.clone()
        D.paged_attention(q.cuda(), *pool.args, q_start=torch.tensor(starts, dtype=torch.int32).cuda(), causal=causal, out=out)
        check(out, ref, tol, keep)
        # with the caller's bounds: the same numbers wherever the bounds change nothing in the split, right ones anyway
        out = keep.clone()
        D.paged_attention(q.cuda(), *pool.args, q_start=torch.tensor(starts, dtype=torch.int32).cuda(), causal=causal, out=out,
                          max_q=max(news), max_kv=max(lens))
        check(out, ref, tol, keep)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("page", [8, 16, 128, 1024])
@pytest.mark.parametrize("n,length,heads,kv_heads", [(1, 5003, 8, 1), (4, 2050, 16, 2), (40, 3001, 4, 2), (16, 999, 32, 8)])
def test_attention_splits_long_caches(dtype, page, n, length, heads, kv_heads):
    pool = Pool([length, length // 3], kv_heads, 128, page, dtype, seed=page)
    q = (2 * torch.randn(2 * n, heads, 128, generator=torch.Generator().manual_seed(1))).to(dtype)
    ref, tol = reference(q, pool.dense, [0, n], [n, n], True, 128 ** -0.5)
    check(D.paged_attention(q.cuda(), *pool.args), ref, tol)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,heads,kv_heads", [(3, 16, 2), (8, 8, 2), (1, 32, 1)])
def test_rows_for_two_column_tiles(dtype, dim, n, heads, kv_heads):
    """17 to 32 rows a key head, lengths around the tiles' and the waves' turns"""
    lens = [n, 15, 16, 33, 64, 65, 127, 129, 300]
    pool = Pool([max(n, x) for x in lens], kv_heads, dim, 8, dtype)
    lens = pool.lens.tolist()
    q = (2 * torch.randn(n * len(lens), heads, dim, generator=torch.Generator().manual_seed(1))).to(dtype)
    for causal in (True, False):
        ref, tol = reference(q, pool.dense, [i * n for i in range(len(lens))], [n] * len(lens), causal, dim ** -0.5)
        check(D.paged_attention(q.cuda(), *pool.args, causal=causal), ref, tol)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_chunks_that_fill_the_card(dtype, dim):
    """enough long chunks for 256-row tiles; 24 tokens of each, the first and the last among them, against 64 bits"""
    news, lens, heads, kv_heads = [1100, 1301], [1500, 1301], 64, 64
    pool = Pool(lens, kv_heads, dim, 64, dtype)
    starts = starts_of(news)
    g = torch.Generator().manual_seed(3)
    q = (2 * torch.randn(starts[-1], heads, dim, generator=g)).to(dtype)
    out = D.paged_attention(q.cuda(), *pool.args, q_start=torch.tensor(starts, dtype=torch.int32).cuda()).cpu()
    for s in range(2):
        for i in [0, news[s] - 1] + torch.randint(0, news[s], (22,), generator=g).tolist():
            k, v = pool.dense[s][:, :lens[s] - news[s] + 1 + i]
            ref, tol = reference(q[starts[s] + i][None], [(k, v)], [0], [1], True, dim ** -0.5)
            check(out[starts[s] + i][None], ref, tol)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("n", [1, 40])
def test_a_long_tail_of_small_weights_counts(dtype, n):
    """one key that outweighs every other by e^17 and 60 000 others: together 0.25 % of the weight, each of them below the
    smallest number fp16 has"""
    length, dim = 60000, 64
    pool = Pool([length], 1, dim, 64, dtype)
    k, v = torch.zeros(length, 1, dim), torch.ones(length, 1, dim)
    k[7, 0, 0], v[7] = 17.0, 0.0
    for j in range(-(-length // 64)):
        pg, rows = int(pool.table[0, j]), slice(j * 64, min(length, j * 64 + 64))
        m = rows.stop - rows.start
        pool.k[pg, :, :m], pool.v[pg, :, :m] = k[rows].transpose(0, 1).to(dtype).cuda(), v[rows].transpose(0, 1).to(dtype).cuda()
    q = torch.zeros(n, 1, dim)
    q[:, 0, 0] = 1.0
    q = q.to(dtype)
    ref, tol = reference(q, [(k.double(), v.double())], [0], [n], True, 1.0)
    assert 0.002 < ref.max() < 0.003
    check(D.paged_attention(q.cuda(), *pool.args, scale=1.0), ref, tol)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("heads", [20, 33, 71])
def test_many_heads_on_one_key_head(dtype, heads):
    """groups of no even size, up to more rows in one token than the thin kernel takes"""
    news, lens = [1, 3, 1, 0, 6], [40, 3, 700, 9, 129]
    pool = Pool(lens, 1, 128, 32, dtype)
    starts = starts_of(news)
    q = (2 * torch.randn(starts[-1], heads, 128, generator=torch.Generator().manual_seed(1))).to(dtype)
    ref, tol = reference(q, pool.dense, starts, news, True, 128 ** -0.5)
    qs = torch.tensor(starts, dtype=torch.int32).cuda()
    check(D.paged_attention(q.cuda(), *pool.args, q_start=qs), ref, tol)
    check(D.paged_attention(q.cuda(), *pool.args, q_start=qs, max_q=6, max_kv=700), ref, tol)
    one = q[:5]
    ref, tol = reference(one, pool.dense, list(range(5)), [1] * 5, True, 128 ** -0.5)
    check(D.paged_attention(one.cuda(), *pool.args), ref, tol)


@gpu
@pytest.mark.parametrize("seqs", [64, 65, 150])
@pytest.mark.parametrize("long_ones", [3, 60])
def test_many_sequences_of_mixed_lengths(seqs, long_ones):
    """single tokens, empty ones and chunks side by side, more sequences than a wave has lanes; few long ones (both kernels, a
    launch each) and many (the tiles take the single tokens along)"""
    rng = random.Random(seqs)
    news = [rng.choice([0, 1, 1, 1, 2]) for _ in range(seqs)]
    for i in rng.sample(range(seqs), long_ones):
        news[i] = rng.randint(20, 90)
    lens = [n + rng.choice([0, 5, 33, 200]) for n in news]
    pool = Pool(lens, 2, 64, 16, torch.bfloat16)
    starts = starts_of(news)
    q = torch.randn(starts[-1], 8, 64, generator=torch.Generator().manual_seed(1)).bfloat16()
    ref, tol = reference(q, pool.dense, starts, news, True, 0.125)
    check(D.paged_attention(q.cuda(), *pool.args, q_start=torch.tensor(starts, dtype=torch.int32).cuda()), ref, tol)
    q = torch.randn(9 * seqs, 8, 64, generator=torch.Generator().manual_seed(2)).bfloat16()
    ref, tol = reference(q, pool.dense, [9 * i for i in range(seqs)], [9] * seqs, True, 0.125)
    check(D.paged_attention(q.cuda(), *pool.args), ref, tol)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])
def test_strided_and_unaligned_rows(dtype):
    """queries, new keys / values and outputs as slices of a packed projection, at offsets that no vector load allows"""
    pool = Pool([30, 45], 2, 64, 16, dtype)
    g = torch.Generator().manual_seed(2)
    packed = torch.randn(10, 3 * 4 * 64 + 5, generator=g).to(dtype).cuda()
    q = packed[:, 3:3 + 256].unflatten(1, (4, 64))
    ref, tol = reference(q.cpu(), pool.dense, [0, 5], [5, 5], True, 0.125)
    out = torch.zeros(10, 4 * 64 + 7, dtype=dtype, device="cuda")
    D.paged_attention(q, *pool.args, out=out[:, 1:257].unflatten(1, (4, 64)))
    check(out[:, 1:257].unflatten(1, (4, 64)), ref, tol)
    assert (out[:, 0] == 0).all() and (out[:, 257:] == 0).all()
    k_new, v_new = packed[:, 259:387].unflatten(1, (2, 64)), packed[:, 390:518].unflatten(1, (2, 64))
    D.paged_append(k_new, v_new, *pool.args)
    for s, n in ((0, 30), (1, 45)):
        for i in range(5):
            pos = n - 5 + i
            pg = int(pool.table[s, pos // 16])
            assert torch.equal(pool.k[pg, :, pos % 16], k_new[s * 5 + i]) and torch.equal(pool.v[pg, :, pos % 16], v_new[s * 5 + i])


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n", [3, 50, 200])
def test_nonfinite_values_behind_the_mask_do_not_leak(dtype, n):
    """infinities and NaN in keys and values that a query does not see (later tokens of its own chunk) leave it alone; those
    that see an infinite value get it"""
    heads, dim, length = 4, 64, n + 37
    pool = Pool([length], 2, dim, 16, dtype, seed=n)
    q = torch.randn(n, heads, dim, generator=torch.Generator().manual_seed(3)).to(dtype)
    ref, tol = reference(q, pool.dense, [0], [n], True, dim ** -0.5)
    cut = n - 1                                                       # the last token's key and value are poisoned
    pg, slot = int(pool.table[0, (length - 1) // 16]), (length - 1) % 16
    for bad in (float("nan"), float("inf"), float("-inf")):
        pool.v[pg, :, slot, ::3] = bad
        out = D.paged_attention(q.cuda(), *pool.args)
        check(out[:cut], ref[:cut], tol[:cut])
        last = out[cut].float()
        assert not torch.isfinite(last[:, ::3]).any() and torch.isfinite(last[:, 1::3]).all()
    pool.k[pg, :, slot] = float("nan")
    out = D.paged_attention(q.cuda(), *pool.args)
    check(out[:cut], ref[:cut], tol[:cut])
    assert torch.isnan(out[cut]).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("n", [1, 60])
def test_bad_numbers_from_the_device(dtype, n):
    """page numbers outside the cache, lengths beyond the table or the caller's bound: NaN for that sequence (for a bad
    page: for the tokens that need it), right results for its neighbours, and an append that drops what has no place"""
    lens = [90, 90, 90, 90]
    pool = Pool(lens, 2, 64, 16, dtype, table_ld=6)
    q = torch.randn(4 * n, 4, 64, generator=torch.Generator().manual_seed(4)).to(dtype)
    ref, tol = reference(q, pool.dense, [i * n for i in range(4)], [n] * 4, True, 0.125)
    table, lens_d = pool.dev_table.clone(), pool.dev_lens.clone()
    for value in (-1, pool.k.shape[0], 2 ** 31 - 1):
        table.copy_(pool.dev_table)
        table[1, 2] = value
        out = D.paged_attention(q.cuda(), pool.k, pool.v, table, pool.dev_lens)
        need = max(0, 32 - (90 - n))                                  # the first token that sees position 32
        assert torch.isnan(out[n + need:2 * n]).all()
        for s in (0, 2, 3):
            check(out[s * n:(s + 1) * n], ref[s * n:(s + 1) * n], tol[s * n:(s + 1) * n])
    for value in (-5, 97, 2 ** 31 - 1):
        lens_d.copy_(pool.dev_lens)
        lens_d[2] = value
        out = D.paged_attention(q.cuda(), pool.k, pool.v, pool.dev_table, lens_d)
        assert torch.isnan(out[2 * n:3 * n]).all()
        check(out[:2 * n], ref[:2 * n], tol[:2 * n])
        check(out[3 * n:], ref[3 * n:], tol[3 * n:])
    out = D.paged_attention(q.cuda(), *pool.args, max_kv=89)
    assert torch.isnan(out).all()
    table.copy_(pool.dev_table)
    table[0, 5] = -1
    before = pool.k.clone()
    new = torch.ones(4, 2, 64, dtype=dtype, device="cuda")
    D.paged_append(new, new, pool.k, pool.v, table, pool.dev_lens)
    changed = (pool.k != before) & ~(torch.isnan(pool.k) & torch.isnan(before))
    touched = changed.flatten(1).any(1).nonzero().flatten().tolist()
    assert sorted(touched) == sorted(int(pool.table[s, 5]) for s in (1, 2, 3))


@gpu
def test_too_many_rows_for_the_bound():
    pool = Pool([60, 60], 2, 64, 16, torch.bfloat16)
    starts = torch.tensor([0, 40, 41], dtype=torch.int32).cuda()
    q = torch.randn(41, 4, 64, generator=torch.Generator().manual_seed(4)).bfloat16()
    out = D.paged_attention(q.cuda(), *pool.args, q_start=starts, max_q=1)
    assert torch.isnan(out[:40]).all()
    ref, tol = reference(q, pool.dense, [0, 40], [40, 1], True, 0.125)
    check(out[40:], ref[40:], tol[40:])


@gpu
def test_offsets_past_32_bits():
    """a cache of more than 2^31 elements per tensor, the sequence in its last pages"""
    page, heads, dim = 1024, 8, 256
    num = 2 ** 31 // (page * heads * dim) + 3
    small = Pool([1500], heads, dim, page, torch.bfloat16)
    k, v = (torch.empty(num, heads, page, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.tensor([[num - 1, num - 2]], dtype=torch.int32)
    for j in range(2):
        k[int(table[0, j])] = small.k[int(small.table[0, j])]
        v[int(table[0, j])] = small.v[int(small.table[0, j])]
    for n in (1, 70):
        q = torch.randn(n, 16, dim, generator=torch.Generator().manual_seed(6)).bfloat16()
        ref, tol = reference(q, small.dense, [0], [n], True, dim ** -0.5)
        check(D.paged_attention(q.cuda(), k, v, table.cuda(), small.dev_lens), ref, tol)
    new = torch.randn(1, heads, dim, device="cuda").bfloat16()
    D.paged_append(new, new, k, v, table.cuda(), small.dev_lens)
    assert torch.equal(k[num - 2, :, 1499 - 1024], new[0]) and torch.equal(v[num - 2, :, 1499 - 1024], new[0])


@gpu
@pytest.mark.parametrize("n,lens", [(1, [70, 2100]), (60, [200, 700])])
def test_captured_and_concurrent_calls(n, lens):
    """one call captured, replayed with other contents and lengths between eager work; two captured graphs and two streams at
    once: every result that of the eager call"""
    pool = Pool(lens, 2, 128, 16, torch.bfloat16, table_ld=150)
    g = torch.Generator().manual_seed(8)
    qs = [torch.randn(2 * n, 8, 128, generator=g).bfloat16().cuda() for _ in range(3)]
    expect = [D.paged_attention(x, *pool.args) for x in qs]
    statics = [torch.empty_like(qs[0]) for _ in range(2)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for st in statics:
            st.copy_(qs[0])
            D.paged_attention(st, *pool.args)
    torch.cuda.current_stream().wait_stream(side)
    for st in statics:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(D.paged_attention(st, *pool.args))
        graphs.append(gr)
    for i in range(6):
        for j, st in enumerate(statics):
            st.copy_(qs[(i + j) % 3])
        torch.cuda.synchronize()
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        with torch.cuda.stream(a):
            graphs[0].replay()
        with torch.cuda.stream(b):
            graphs[1].replay()
        torch.cuda.synchronize()
        for j in range(2):
            assert torch.equal(outs[j], expect[(i + j) % 3])
        D.paged_attention(qs[2], *pool.args)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got.append((i, D.paged_attention(qs[i % 3], *pool.args)))
    torch.cuda.synchronize()
    for i, o in got:
        assert torch.equal(o, expect[i % 3])


@gpu
def test_empty_calls():
    pool = Pool([0, 0], 2, 64, 16, torch.float32)
    assert D.paged_attention(torch.zeros(0, 4, 64).cuda(), *pool.args).shape == (0, 4, 64)
    out = D.paged_attention(torch.ones(2, 4, 64).cuda(), *pool.args)
    assert (out == 0).all()
    D.paged_append(torch.ones(2, 2, 64).cuda(), torch.ones(2, 2, 64).cuda(), *pool.args)       # no position: dropped
    none = [pool.k, pool.v, pool.dev_table[:0], pool.dev_lens[:0]]
    keep = torch.full((3, 4, 64), 5.0).cuda()
    D.paged_attention(torch.zeros(3, 4, 64).cuda(), *none, q_start=torch.zeros(1, dtype=torch.int32).cuda(), out=keep)
    assert (keep == 5).all()


# ---------------------------------------------------------------------------------------------------- GPU: selection
def select_reference(logits, scores, finished, eos, n):
    x = logits.double().cpu()
    b, k, v = x.shape
    s = scores.double().cpu()
    cand = torch.full((b, k, v), float("-inf"), dtype=torch.float64)
    for i in range(b):
        for j in range(k):
            if not math.isfinite(s[i, j]):
                continue
            if finished is not None and bool(finished[i, j]):
                cand[i, j, eos] = s[i, j]
                continue
            norm = torch.logsumexp(x[i, j], 0)
            if math.isfinite(norm):
                cand[i, j] = torch.nan_to_num(s[i, j] + (x[i, j] - norm), nan=float("-inf"), neginf=float("-inf"))
    val, idx = torch.sort(cand.view(b, -1), dim=1, descending=True, stable=True)
    parents, tokens = idx[:, :n] // v, idx[:, :n] % v
    fin = tokens == eos
    if finished is not None:
        fin |= torch.gather(finished.cpu(), 1, parents)
    return val[:, :n], parents.int(), tokens, fin


def check_select(logits, scores, finished=None, eos=None, n=None):
    n = scores.shape[1] if n is None else n
    val, par, tok, fin = select_reference(logits, scores, finished, eos if eos is not None else -1, n)
    got = D.beam_select(logits.cuda(), scores.cuda(), None if finished is None else finished.cuda(), eos=eos, n=n)
    assert torch.equal(got[1].cpu(), par) and torch.equal(got[2].cpu(), tok) and torch.equal(got[3].cpu(), fin)
    # one rounding to fp32, and 2^-30 for the normaliser
    ok = (got[0].cpu().double() - val).abs() <= val.abs() * 2.0 ** -24 + 2.0 ** -30
    assert (ok | (got[0].cpu().double() == val)).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("batch,beams,vocab,n", [(1, 1, 1, 1), (1, 1, 5, 5), (3, 4, 7, 4), (2, 3, 63, 6), (5, 5, 65, 5), (2, 8, 2047, 8),
                                                 (4, 4, 2049, 8), (2, 4, 6625, 4), (1, 4, 50001, 4), (3, 16, 4097, 16), (1, 64, 301, 64),
                                                 (2, 2, 131073, 2), (70, 2, 999, 2)])
def test_selection_against_64_bits(dtype, batch, beams, vocab, n):
    g = torch.Generator().manual_seed(vocab)
    x = (3 * torch.randn(batch, beams, vocab, generator=g)).to(dtype)
    s = -5 * torch.rand(batch, beams, generator=g)
    check_select(x, s, n=n)
    fin = torch.rand(batch, beams, generator=g) < 0.4
    check_select(x, s, fin, eos=vocab // 2, n=n)
    s[:, 1:] = float("-inf")                                          # a search's first step
    check_select(x, s, n=n)


@gpu
@pytest.mark.parametrize("vocab", [9, 700, 9001])
def test_selection_ties_masks_and_nonfinite(vocab):
    g = torch.Generator().manual_seed(1)
    s = torch.zeros(2, 3)
    check_select(torch.zeros(2, 3, vocab), s, n=7)                    # everything equal: the lowest indices
    x = torch.randint(0, 3, (2, 3, vocab), generator=g).float()
    x[:, 1] = x[:, 0]
    x[:, 2] = x[:, 0]
    check_select(x, s, n=9)                                           # equal beams: the lower beam first
    x = torch.randn(2, 3, vocab, generator=g)
    x[0, :, 4:] = float("-inf")                                       # a masked vocabulary: fewer live ones than asked for
    x[1, 1] = float("-inf")                                           # a beam with nothing left
    check_select(x, s, n=9)
    check_select(x, s, n=20)
    x = torch.randn(2, 3, vocab, generator=g)
    x[0, 1, 3] = float("nan")
    x[1, 2, 0] = float("inf")
    check_select(x, s, n=9)
    s = torch.tensor([[0.0, float("nan"), -1.0], [float("-inf")] * 3])
    check_select(torch.randn(2, 3, vocab, generator=g), s, n=9)
    fin = torch.tensor([[True, True, True], [True, False, True]])
    check_select(torch.randn(2, 3, vocab, generator=g), s, fin, eos=0, n=9)
    x = torch.full((2, 3, vocab), torch.finfo(torch.float32).min)     # masks of the type's lowest value
    x[:, :, 5] = 1.0
    check_select(x, torch.tensor([[-1.0, -2.0, -3.0]] * 2), n=5)
    z = torch.zeros(1, 2, vocab)
    z[0, 0, 1::2] = -0.0                                              # both zeros are one value
    check_select(z, torch.zeros(1, 2), n=6)
    up = torch.arange(vocab).float().expand(2, 3, vocab).contiguous() / 64
    check_select(up, torch.zeros(2, 3), n=9)                          # ever better ones to the end


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("beams", [2, 20])
def test_selection_at_the_ends_of_rows(dtype, beams):
    """rows shorter than a 16-byte word, rows that end inside one, and rows that start at any element of one"""
    for vocab in (1, 2, 3, 4, 5, 7, 8, 9, 15, 17, 255, 257, 511, 513, 2045, 2051, 8189, 8195, 14337):
        g = torch.Generator().manual_seed(vocab)
        n = min(beams * vocab, 11)
        x = torch.randn(2, beams, vocab, generator=g).to(dtype)
        x[:, :, vocab // 2:] += 2                                     # the best ones near the ends
        s = -torch.rand(2, beams, generator=g)
        check_select(x, s, n=n)
        wide = torch.full((2, beams, vocab + 6), float("nan"), dtype=dtype)      # neighbours of a row that must not count
        wide[:, :, 3:3 + vocab] = x
        val, par, tok, fin = select_reference(x, s, None, -1, n)
        got = D.beam_select(wide.cuda()[:, :, 3:3 + vocab], s.cuda(), n=n)
        assert torch.equal(got[1].cpu(), par) and torch.equal(got[2].cpu(), tok), vocab
        assert torch.isfinite(got[0]).all()


@gpu
@pytest.mark.parametrize("n", [1, 16, 17, 64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_selection_of_many_equal_candidates(dtype, n):
    """more values of one size than a wave's buffer holds: among the best ones, as the mask's value, everywhere, in either order"""
    g = torch.Generator().manual_seed(n)
    s = torch.tensor([[0.0, -0.5, -1.0]])
    for vocab in (600, 20000, 70001):
        x = torch.randn(1, 3, vocab, generator=g).clamp_max(0.5).to(dtype)
        check_select(x, s, n=n)                                       # a third of them the maximum
        for live in (1, 5, 40):                                       # a vocabulary masked to a few tokens
            y = torch.full_like(x, float("-inf"))
            y[:, :, torch.randperm(vocab, generator=g)[:live]] = 1.5
            check_select(y, s, n=n)
            check_select(torch.where(y == 1.5, x, torch.full_like(x, torch.finfo(dtype).min)), s, n=n)
        check_select(torch.randint(0, 2, (1, 3, vocab), generator=g).to(dtype), s, n=n)
        steps = (torch.arange(vocab) // 37).float().expand(1, 3, vocab) / 1024      # rising and falling in long steps
        check_select(steps.to(dtype).contiguous(), s, n=n)
        check_select(steps.flip(2).to(dtype).contiguous(), s, n=n)


@gpu
def test_selection_separates_neighbours_in_64_bits():
    """two beams whose candidates differ by less than fp32 resolves at that magnitude"""
    x = torch.randn(1, 2, 500, generator=torch.Generator().manual_seed(3))
    x[0, 1] = x[0, 0]
    x[0, 1, 17] += 4e-5                                               # raises one logit: every other token falls behind
    x[0, 0, 400], x[0, 1, 400] = 9.0, 9.0
    check_select(x, torch.full((1, 2), -30.0), n=8)


@gpu
def test_selection_of_strided_logits_streams_and_graphs():
    g = torch.Generator().manual_seed(2)
    big = torch.randn(4, 3, 1003, generator=g)
    view = big[:, :, 1:1000]
    s = -torch.rand(4, 3, generator=g)
    val, par, tok, fin = select_reference(view, s, None, -1, 3)
    d = big.cuda()[:, :, 1:1000]
    got = D.beam_select(d, s.cuda())
    assert torch.equal(got[1].cpu(), par) and torch.equal(got[2].cpu(), tok)
    last = torch.randn(4, 3, 7, 999, generator=g)                     # the last position of a prompt's logits
    val, par, tok, fin = select_reference(last[:, :, -1], s, None, -1, 3)
    got = D.beam_select(last.cuda()[:, :, -1], s.cuda())
    assert torch.equal(got[1].cpu(), par) and torch.equal(got[2].cpu(), tok)
    for vocab in (999, 70001):
        xs = [torch.randn(2, 4, vocab, generator=g).cuda() for _ in range(3)]
        sc = (-torch.rand(2, 4, generator=g)).cuda()
        want = [D.beam_select(x, sc) for x in xs]
        st = xs[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            D.beam_select(st, sc)
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = D.beam_select(st, sc)
        for i in range(5):
            st.copy_(xs[i % 3])
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(res, want[i % 3]))
            D.beam_select(xs[(i + 1) % 3], sc)


# --------------------------------------------------------------------------------------------------- GPU: reordering
@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("groups,beams,heads,dim,page,layers", [(1, 1, 1, 64, 8, 1), (3, 4, 4, 256, 16, 1), (2, 5, 3, 64, 128, 40),
                                                                (4, 8, 2, 128, 32, 2)])
@pytest.mark.parametrize("length", [0, 1, 15, 16, 31, 127, 128, 300])
def test_reorder_against_a_plain_form(dtype, groups, beams, heads, dim, page, layers, length):
    g = torch.Generator().manual_seed(length)
    slots, per = groups * beams, 300 // page + 2
    num = slots * (per + 1)
    perm = torch.randperm(num, generator=g).to(torch.int32)
    table, spare = perm[:slots * per].view(slots, per).clone(), perm[slots * per:].clone()
    lens = torch.full((slots,), length, dtype=torch.int32)
    if groups > 1:
        lens[beams:] = max(0, length - 3)
    parents = torch.randint(0, beams, (groups, beams), generator=g).to(torch.int32)
    parents[0, -1] = 99 if beams > 1 else 0                           # no such beam: it stays what it is
    pages = [torch.randn(num, heads, page, dim, generator=g).to(dtype) for _ in range(2 * layers)]
    dev = [p.cuda() for p in pages]
    t2, s2 = D.beam_reorder(parents.cuda(), table.cuda(), lens.cuda(), spare.cuda(), dev)
    want_t, want_s = table.clone(), spare.clone()
    want_p = [p.clone() for p in pages]
    for j in range(slots):
        p = int(parents.view(-1)[j])
        src = j // beams * beams + p if 0 <= p < beams else j
        n = int(lens[j])
        want_t[j, :n // page] = table[src, :n // page]
        if n % page and src != j:
            want_t[j, n // page], want_s[j] = spare[j], table[j, n // page]
            for a, b in zip(want_p, pages):
                a[spare[j], :, :n % page] = b[table[src, n // page], :, :n % page]
    assert torch.equal(t2.cpu(), want_t) and torch.equal(s2.cpu(), want_s)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, want_p))
    # in place
    dev = [p.cuda() for p in pages]
    t, s = table.cuda(), spare.cuda()
    D.beam_reorder(parents.cuda(), t, lens.cuda(), s, dev, t, s)
    assert torch.equal(t.cpu(), want_t) and torch.equal(s.cpu(), want_s)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, want_p))


@gpu
def test_reorder_with_bad_numbers_reads_and_writes_nothing_outside():
    table = torch.tensor([[0, -4], [3, 10 ** 9]], dtype=torch.int32).cuda()
    spare = torch.tensor([4, 2 ** 31 - 1], dtype=torch.int32).cuda()
    parents = torch.tensor([[1, 0]], dtype=torch.int32).cuda()
    for length in (20, -3, 33, 2 ** 31 - 1):
        pages = [torch.randn(6, 2, 16, 64).cuda()]
        before = pages[0].clone()
        lens = torch.tensor([length, length], dtype=torch.int32).cuda()
        t, s = D.beam_reorder(parents, table, lens, spare, pages)
        assert torch.equal(pages[0], before)
        if length != 20:
            assert torch.equal(t, table) and torch.equal(s, spare)


# ------------------------------------------------------------------------------------------------ GPU: used together
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_search_steps_equal_dense_caches(dtype):
    """40 steps of a beam search with random survivors: append, attend, reorder on pages against dense per-beam caches that
    are copied whole"""
    groups, beams, heads, kv_heads, dim, page = 3, 4, 4, 2, 64, 8
    slots = groups * beams
    g = torch.Generator().manual_seed(11)
    cache = D.PagedCache(slots, 40, kv_heads, dim, layers=2, page=page, dtype=dtype)
    dense = [[torch.zeros(2, 0, kv_heads, dim, dtype=torch.float64) for _ in range(slots)] for _ in range(2)]
    for step in range(40):
        cache.advance(1)
        for layer in range(2):
            k, v = (torch.randn(slots, kv_heads, dim, generator=g).to(dtype) for _ in range(2))
            q = torch.randn(slots, heads, dim, generator=g).to(dtype)
            cache.append(layer, k.cuda(), v.cuda())
            for s in range(slots):
                dense[layer][s] = torch.cat([dense[layer][s], torch.stack([k[s], v[s]]).double()[:, None]], 1)
            ref, tol = reference(q, dense[layer], list(range(slots)), [1] * slots, True, dim ** -0.5)
            check(cache.attend(layer, q.cuda()), ref, tol)
        parents = torch.randint(0, beams, (groups, beams), generator=g).to(torch.int32)
        cache.reorder(parents.cuda())
        for layer in range(2):
            dense[layer] = [dense[layer][s // beams * beams + int(parents.view(-1)[s])] for s in range(slots)]
    owned = torch.cat([cache.table.flatten(), cache.spare]).unique()
    assert owned.numel() >= slots                                     # no spare page was lost on the way


# ---------------------------------------------------------------------------------------------- GPU: the recognizers
def _recognizer(kind):
    from fudanocr_amd.utils.weight_fill import fill_module_
    if kind == "strokes":
        from fudanocr_amd.sld.model.transformer import Transformer
        m = Transformer("stroke")
    elif kind == "characters":
        from fudanocr_amd.loss.transformer import Transformer
        m = Transformer()
    else:
        from fudanocr_amd.loss.transformer_english_decomposition import Transformer
        m = Transformer()
    fill_module_(m)
    return m.cuda().eval()


def _dense_logits(model, kind, image, tokens):
    """[N, L, vocab] by the models' own forward on whole prefixes"""
    with torch.no_grad():
        if kind == "strokes":
            length = torch.full((tokens.shape[0],), tokens.shape[1])
            return model(image, length, tokens, test=True)["pred"]
        return model.forward_padded(image, tokens)[0]


@gpu
@pytest.mark.parametrize("kind,channels,width", [("strokes", 3, 32), ("characters", 1, 128), ("english_strokes", 4, 128)])
@pytest.mark.parametrize("beams", [1, 3])
def test_recognizers_beam_search_equals_whole_prefixes(kind, channels, width, beams):
    """the cached search against the same search by whole prefixes through the model's own forward and a 64-bit selection on
    the CPU.  The two sum in another order, so scores agree to fp32 products over the network (1e-3 relative) and a hypothesis may
    differ only where the dense search has one of the same score."""
    model = _recognizer(kind)
    g = torch.Generator().manual_seed(5)
    batch, steps = 3, 20                                              # past a page of 16 tokens
    image = (torch.rand(batch, channels, 32, width, generator=g) * 2 - 1).cuda()
    tokens, scores = model.beam_search(image, beams=beams, max_len=steps)
    assert tokens.shape == (batch, beams, steps) and scores.shape == (batch, beams)
    assert (scores[:, :-1] >= scores[:, 1:]).all()
    start, eos = (0, 6) if kind == "strokes" else (0, 0)
    ended = (tokens == eos).int().cummax(-1).values.bool()
    assert (tokens[ended] == eos).all()                               # nothing but eos behind the first one
    # a hypothesis' score is the sum of its tokens' log-probabilities, by the dense forward
    rep = image.repeat_interleave(beams, 0)
    flat = tokens.view(-1, steps)
    prefix = torch.cat([torch.full_like(flat[:, :1], start), flat[:, :-1]], 1)
    logp = torch.log_softmax(_dense_logits(model, kind, rep, prefix).double(), -1)
    per = torch.gather(logp, 2, flat[..., None])[..., 0]
    live = torch.cat([torch.ones_like(ended.view(-1, steps)[:, :1]), ~ended.view(-1, steps)[:, :-1]], 1)
    want = (per * live).sum(1).view(batch, beams)
    ok = torch.isfinite(scores)
    assert ok[:, 0].all() and ((scores.double() - want).abs() <= 1e-3 * (1 + want.abs()))[ok].all()
    # the dense search, beam by beam
    beam_scores = torch.full((batch, beams), float("-inf"), dtype=torch.float32)
    beam_scores[:, 0] = 0
    done = torch.zeros(batch, beams, dtype=torch.bool)
    seqs = torch.full((batch, beams, 1), start)
    for _ in range(steps):
        lg = _dense_logits(model, kind, rep, seqs.view(batch * beams, -1).cuda())[:, -1].view(batch, beams, -1).cpu()
        val, par, tok, fin = select_reference(lg, beam_scores, done, eos, beams)
        seqs = torch.cat([torch.gather(seqs, 1, par.long()[..., None].expand(-1, -1, seqs.shape[2])), tok[..., None]], 2)
        beam_scores, done = val.float(), fin
    assert (beam_scores - scores.cpu()).abs().max() <= 1e-3 * (1 + beam_scores.abs().max())
    for b in range(batch):
        for j in range(beams):
            if not torch.equal(seqs[b, j, 1:], tokens[b, j].cpu()):
                close = (beam_scores[b] - scores[b, j].cpu()).abs() <= 2e-3 * (1 + scores[b, j].abs().item())
                assert int(close.sum()) > 1, (b, j)


@gpu
def test_recognizer_beam_search_refusals():
    model = _recognizer("strokes")
    image = torch.zeros(1, 3, 32, 32).cuda()
    _raises("1 to 64", model.beam_search, image, beams=0)
    _raises("1 to 64", model.beam_search, image, beams=65)
    _raises("max_len", model.beam_search, image, max_len=7001)
    assert model.beam_search(image, beams=2, max_len=1)[0].shape == (1, 2, 1)
    _raises("eval mode", model.train().beam_search, image)


# ------------------------------------------------------------------------------- refusals of shared memory and of gradients
def test_beam_search_refuses_before_the_encoder_runs():
    """a model in training mode is refused before its encoder could move the batch norms' running statistics"""
    from fudanocr_amd.loss.transformer import Transformer as Characters
    from fudanocr_amd.loss.transformer_english_decomposition import Transformer as EnglishStrokes
    from fudanocr_amd.sld.model.transformer import Transformer as Strokes

    def never(*a, **kw):
        raise AssertionError("the encoder ran")
    for model, image in ((Strokes("stroke"), torch.zeros(1, 3, 32, 32)), (Characters(), torch.zeros(1, 1, 32, 128)),
                         (EnglishStrokes(), torch.zeros(1, 1, 32, 128))):
        model.encoder.forward = never
        _raises("eval mode", model.train().beam_search, image)
        _raises("1 to 64", model.eval().beam_search, image, beams=65)
        _raises("max_len", model.beam_search, image, max_len=0)


def test_whatever_wants_a_gradient_is_refused():
    c, q = _cpu_cache(), torch.zeros(3, 4, 64)
    for i in (0, 1):
        g = list(c)
        g[i] = c[i].clone().requires_grad_(True)
        _raises("wants a gradient", D.paged_attention, q, *g)
        _raises("wants a gradient", D.paged_append, q[:, :2], q[:, :2], *g)
        with torch.no_grad():
            _raises("on the GPU", D.paged_attention, q, *g)
    x, s = torch.zeros(2, 3, 7), torch.zeros(2, 3, requires_grad=True)
    _raises("wants a gradient", D.beam_select, x, s)
    p, t, sp = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(6, 2, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)
    _raises("wants a gradient", D.beam_reorder, p, t, sp, sp, [torch.zeros(8, 2, 16, 64, requires_grad=True)])
    with torch.no_grad():
        _raises("on the GPU", D.beam_select, x, s)


def test_outputs_whose_rows_overlap_are_refused():
    c, q = _cpu_cache(), torch.zeros(3, 4, 64)
    buf = torch.zeros(4096)
    for strides in ((64, 64, 1), (256, 32, 1), (255, 64, 1), (64, 128, 1), (0, 64, 1), (256, 0, 1)):
        _raises("rows of its own", D.paged_attention, q, *c, out=buf.as_strided((3, 4, 64), strides))
    for strides in ((256, 64, 1), (64, 192, 1), (300, 70, 1)):        # apart: refused for being on the CPU alone
        _raises("on the GPU", D.paged_attention, q, *c, out=buf.as_strided((3, 4, 64), strides))
    _raises("on the GPU", D.paged_attention, q[:1], c[0], c[1], c[2][:1], c[3][:1], out=buf.as_strided((1, 4, 64), (0, 64, 1)))


def test_c_entries_refuse_shared_memory():
    """a result that lies in what is read, as addresses that are never followed: 8 pages x 2 heads x 16 x 64 fp32 = 64 KB"""
    from fudanocr_amd import _lib
    lib = _lib.load()
    size, k, v, far = 65536, 1 << 20, 1 << 21, 1 << 24

    def attend(q, o):
        rc = lib.focr_paged_attention_fwd(q, 256, 64, k, v, far, far, None, o, 256, 64, None, 0, 3, 3, 4, 2, 64, 16, 2, 8, 1, 32, 0.1,
                                          1, 0, None)
        return rc, lib.focr_last_error().decode()

    def append(kn, vn, kp=k, vp=v):
        rc = lib.focr_paged_append(kn, vn, 128, 64, 128, 64, kp, vp, far, far, None, 3, 3, 2, 64, 16, 2, 8, 0, None)
        return rc, lib.focr_last_error().decode()
    rows = 3 * 256 * 4
    for o in (k, k - rows + 16, k + size - 16, v, v + 4096, far + 2 * size + rows - 16, far + 2 * size):
        rc, msg = attend(far + 2 * size, o)
        assert rc == -1 and "share" in msg, (o, rc, msg)
    rows = 3 * 128 * 4
    for a, b in ((k, far), (far, v), (far, k + size - 16), (v - rows + 16, far), (far, k)):
        rc, msg = append(a, b)
        assert rc == -1 and "share" in msg, (a, b, rc, msg)
    rc, msg = append(far, far, k, k + size - 16)
    assert rc == -1 and "share" in msg, (rc, msg)
    import ctypes
    pages = (ctypes.c_void_p * 1)(k)

    def reorder(table, spare, table_out, spare_out):
        rc = lib.focr_beam_reorder(far, table, far, spare, table_out, spare_out, pages, 1, 2, 3, 2, 64, 16, 4, 8, 0, None)
        return rc, lib.focr_last_error().decode()
    t, s = v, v + 4096                                                # 6 x 4 entries = 96 bytes, 6 spares = 24
    for table_out, spare_out in ((t + 16, s), (t - 80, s), (t, s + 4), (t, s - 20), (t, t + 92), (s - 92, s), (far, t), (t, far)):
        rc, msg = reorder(t, s, table_out, spare_out)
        assert rc == -1 and "share" in msg, (table_out, spare_out, rc, msg)


# ------------------------------------------------------------------------------------------ fp32 sums under a moving maximum
def _shared_pages(k, v, seqs, page):
    """one sequence's keys and values [length, heads, dim] as a cache that all of `seqs` sequences read"""
    length, heads, dim = k.shape
    per = length // page
    pages = [x.view(per, page, heads, dim).transpose(1, 2).contiguous().cuda() for x in (k, v)]
    table = torch.arange(per, dtype=torch.int32).expand(seqs, per).contiguous().cuda()
    return (*pages, table, torch.full((seqs,), length, dtype=torch.int32).cuda())


@gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n", [12, 32, 40])
@pytest.mark.parametrize("top", [299.0, 301.0, 407.0])
def test_fp32_rows_whose_maximum_stands_are_not_rescaled(dim, n, top):
    """One row of a wave finds a new maximum every 16 keys, the others have the same score everywhere: all their weights are 1,
    their sums whole numbers, and the half of the values that is 1 gives 1/2 up to the last division (two roundings).  Rows for both
    forms of the thin kernel and for the tiles; heads and sequences enough that a block has a long run of keys."""
    length, heads, seqs = 4096, 64, 8
    k, v = torch.zeros(length, 1, dim), torch.zeros(length, 1, dim)
    k[:, 0, 0] = (torch.arange(length) // 16).float()
    k[:, 0, 1] = top
    v[:length // 2] = 1.0
    q = torch.zeros(seqs * n, heads, dim)
    q[:, :, 1] = 1.0
    q[::n, :, 1], q[::n, :, 0] = 0.0, 1.0
    args = _shared_pages(k.expand(length, heads, dim), v.expand(length, heads, dim), seqs, 64)
    out = D.paged_attention(q.cuda(), *args, causal=False, scale=1.0).cpu().view(seqs, n, heads, dim)
    assert (out[:, 1:] - 0.5).abs().max() <= 2.0 ** -24
    ref, tol = reference(q[:1, :1], [(k.double(), v.double())], [0], [1], False, 1.0)
    check(out[:1, 0, :1], ref, tol)
    assert torch.equal(out[:, 0], out[:1, 0, :1].expand(seqs, heads, dim))


@gpu
@pytest.mark.parametrize("n", [1, 20, 40])
@pytest.mark.parametrize("top", [299.0, 300.0, 301.0, 407.0, 1000.5])
def test_fp32_parts_join_by_the_difference_of_their_maxima(n, top):
    """a long axis in parts, half of them with a maximum one lower than the others': a / (a + b / e).  The lower weight is off by the
    rounding of c and of the argument (log2 e each, half a step, times ln 2) and a step of the exponential, together 2^-22;
    the up to 16 parts are added one after the other in numerator and denominator, half a step each, and divided."""
    length, dim = 4096, 64
    k, v = torch.zeros(length, 1, dim), torch.zeros(length, 1, dim)
    k[:, 0, 0] = top - (torch.arange(length) >= length // 2).float()
    v[:length // 2] = 1.0
    q = torch.zeros(n, 1, dim)
    q[:, 0, 0] = 1.0
    out = D.paged_attention(q.cuda(), *_shared_pages(k, v, 1, 64), causal=False, scale=1.0).cpu().double()
    want = 1.0 / (1.0 + math.exp(-1.0))
    assert (out - want).abs().max() <= want * (2.0 ** -22 + 33 * 2.0 ** -24)


@gpu
@pytest.mark.parametrize("n", [32, 64])
def test_fp32_error_over_a_long_axis_is_that_of_random_roundings(n):
    """16 384 keys, scores of deviation 2: relative to the output's size the error of a row is, in the mean square, that of independent
    roundings -- of the dim partial sums of a score (5.5e-7), of the argument's difference, product and constant (2.8, 2.8 and
    2.4e-7 at 8 below the maximum), of the exponential (0.6e-7) and of some 700 additions to each of two sums (5.4e-7 each):
    1.1e-6, and at most twice that"""
    length, heads, seqs, dim = 16384, 32, 16, 128
    g = torch.Generator().manual_seed(9)
    k, v = torch.randn(length, heads, dim, generator=g), torch.randn(length, heads, dim, generator=g)
    q = 2 * torch.randn(seqs * n, heads, dim, generator=g)
    out = D.paged_attention(q.cuda(), *_shared_pages(k, v, seqs, 64), causal=False).cpu().double()
    for s, h in ((0, 0), (seqs - 1, heads - 1)):
        rows = slice(s * n, (s + 1) * n)
        want = torch.softmax(q[rows, h].double() @ k[:, h].double().t() * dim ** -0.5, -1) @ v[:, h].double()
        err = (out[rows, h] - want).square().mean(-1).sqrt() / want.square().mean(-1).sqrt()
        assert err.square().mean().sqrt() <= 2.2e-6, float(err.max())


# ------------------------------------------------------------------------------------------- infinite values that a row sees
def _class(x):
    return torch.where(torch.isnan(x), 3, torch.where(x == math.inf, 1, torch.where(x == -math.inf, 2, 0)))


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,length,at", [(3, 3, 1), (50, 50, 2), (50, 50, 40), (300, 300, 5), (300, 300, 200), (50, 1300, 1282),
                                         (50, 1300, 1260), (50, 1300, 700), (9, 1300, 1294)])
def test_rows_that_see_an_infinite_value_get_it(dtype, dim, n, length, at):
    """prompts from their first token on, and the end of a long axis in parts of 256 keys: an infinity in the values goes, with its
    sign, to the rows that see it (a NaN and infinities of both signs make NaN), and to no other"""
    pool = Pool([length], 2, dim, 16, dtype, seed=n)
    k, v = pool.dense[0]
    q = torch.randn(n, 4, dim, generator=torch.Generator().manual_seed(3)).to(dtype)
    ref, tol = reference(q, pool.dense, [0], [n], True, dim ** -0.5)
    for j, row in ((at, [math.inf, -math.inf, math.nan, math.inf]), (at + 1, [0.0, 0.0, 0.0, -math.inf])):
        pool.v[int(pool.table[0, j // 16]), :, j % 16, 5:9] = torch.tensor(row).to(dtype).cuda()
    out = D.paged_attention(q.cuda(), *pool.args, max_kv=length).cpu()
    want = torch.zeros(n, 4, dim, dtype=torch.int64)
    seen = torch.arange(length - n, length)
    for col, cls in ((5, 1), (6, 2), (7, 3)):
        want[seen >= at, :, col] = cls
    want[seen == at, :, 8], want[seen > at, :, 8] = 1, 3
    assert torch.equal(_class(out), want)
    fine = torch.ones(dim, dtype=torch.bool)
    fine[5:9] = False                                                 # (at + 1 has zeros there now)
    check(out[:, :, fine], ref[:, :, fine], tol[:, :, fine])


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n", [3, 50])
def test_infinite_values_where_the_maximum_jumps(dtype, n):
    """the tile that brings an infinite value raises the maximum so far that what came before weighs nothing: the infinity stays"""
    dim, length = 64, 64 + n
    pool = Pool([length], 1, dim, 64, dtype)
    q = torch.zeros(n, 1, dim, dtype=dtype)
    q[:, 0, 0] = 1.0
    page = int(pool.table[0, 1])
    pool.k[int(pool.table[0, 0]), 0], pool.k[page, 0] = 0.0, 0.0
    pool.k[page, 0, 0, 0], pool.k[page, 0, 1, 0] = 200.0, 199.0
    pool.v[page, 0, 1, 9] = math.inf
    out = D.paged_attention(q.cuda(), *pool.args, scale=1.0).cpu()
    want = torch.zeros(n, 1, dim, dtype=torch.int64)
    want[1:, :, 9] = 1                                                # the first of the new tokens does not see it
    assert torch.equal(_class(out), want)


# ------------------------------------------------------------------------------------------------ a cache's step in a graph
@gpu
def test_a_captured_step_of_a_cache_replays_as_the_cache_grows():
    """append, attend and reorder of two layers captured while the cache is nearly empty, replayed to its last token, with eager steps
    in between, against dense caches; `advance` itself is refused inside the capture"""
    groups, beams, heads, kv_heads, dim, page, max_len = 2, 3, 4, 2, 64, 8, 300
    slots = groups * beams
    g = torch.Generator().manual_seed(12)
    cache = D.PagedCache(slots, max_len, kv_heads, dim, layers=2, page=page)
    k, v, q = (torch.zeros(2, slots, h, dim, device="cuda") for h in (kv_heads, kv_heads, heads))
    parents = torch.zeros(groups, beams, dtype=torch.int32, device="cuda")
    dense = [[torch.zeros(2, 0, kv_heads, dim, dtype=torch.float64) for _ in range(slots)] for _ in range(2)]

    def step():
        for layer in range(2):
            cache.append(layer, k[layer], v[layer])
        out = [cache.attend(layer, q[layer]) for layer in range(2)]
        cache.reorder(parents)
        return out
    graph = torch.cuda.CUDAGraph()
    for at in range(max_len):
        cache.advance(1)
        new = [torch.randn(2, slots, h, dim, generator=g) for h in (kv_heads, kv_heads, heads)]
        for dst, src in zip((k, v, q), new):
            dst.copy_(src)
        src = torch.randint(0, beams, (groups, beams), generator=g).to(torch.int32)
        parents.copy_(src)
        if at == 2:
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                _raises("outside the graph", cache.advance, 1)
                captured = step()
        if at < 2 or at % 7 == 0:
            out = step()
        else:
            graph.replay()
            out = captured
        torch.cuda.synchronize()
        for layer in range(2):
            for s in range(slots):
                dense[layer][s] = torch.cat([dense[layer][s], torch.stack([new[0][layer, s], new[1][layer, s]]).double()[:, None]], 1)
            if at < 20 or at % 16 in (0, 1) or at > max_len - 3:
                ref, tol = reference(new[2][layer], dense[layer], list(range(slots)), [1] * slots, True, dim ** -0.5)
                check(out[layer], ref, tol)
            dense[layer] = [dense[layer][s // beams * beams + int(src.view(-1)[s])] for s in range(slots)]
    _raises("in a cache of 300", cache.advance, 1)


# ------------------------------------------------------------------------------------- offsets that run over the rows there are
def test_offsets_that_do_not_fit_on_the_cpu(tmp_path):
    """csrc/paged_index.h on offsets in front of the first row and behind the last, under sanitizers (tests/cpp/paged_offsets_check.cpp)"""
    exe = str(tmp_path / "paged_offsets_check")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-I",
                           os.path.join(ROOT, "fudanocr_amd", "csrc"), os.path.join(ROOT, "tests", "cpp", "paged_offsets_check.cpp"),
                           "-o", exe])
    out = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout[-2000:] + out.stderr[-2000:]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("seqs", [3, 64, 65, 150])
@pytest.mark.parametrize("news", [1, 7, 90])
@pytest.mark.parametrize("heads", [2, 8])
def test_offsets_over_the_first_and_last_row_give_nan(dtype, seqs, news, heads):
    """the first sequence claims rows in front of the tensor, the last ones rows behind it: NaN in the rows of theirs that there are,
    the others' results as they would be, and an append that writes the others' rows alone"""
    lens = [news + 30] * seqs
    pool = Pool(lens, 2, 64, 16, dtype)
    starts = [i * news for i in range(seqs + 1)]
    tokens = starts[seqs - 1] + (news + 1) // 2                       # half of the last sequence is there
    g = torch.Generator().manual_seed(4)
    q = torch.randn(tokens, heads, 64, generator=g).to(dtype)
    ref, tol = reference(q, pool.dense[1:-1], starts[1:-2], [news] * (seqs - 2), True, 0.125)
    for over in (1, 1000, 2 ** 31 - 1 - starts[-1]):
        qs = torch.tensor(starts, dtype=torch.int32)
        qs[0] = -over
        qs[-1] += over
        for kw in ({}, {"max_q": news + 1000, "max_kv": news + 30}):
            out = torch.full((tokens, heads, 64), 7.0, dtype=dtype, device="cuda")
            D.paged_attention(q.cuda(), *pool.args, q_start=qs.cuda(), out=out, **kw)
            assert torch.isnan(out[:news]).all() and torch.isnan(out[starts[-2]:]).all()
            check(out[starts[1]:starts[-2]], ref[starts[1]:starts[-2]], tol[starts[1]:starts[-2]])
    qs[-2] = 2 ** 31 - 2                                              # the last sequence has no rows, the one before it too many
    out = D.paged_attention(q.cuda(), *pool.args, q_start=qs.cuda())
    assert torch.isnan(out[:news]).all() and torch.isnan(out[starts[-3]:]).all()
    check(out[starts[1]:starts[-3]], ref[starts[1]:starts[-3]], tol[starts[1]:starts[-3]])
    before = pool.k.clone()
    new = torch.full((tokens, 2, 64), 3.0, dtype=dtype, device="cuda")
    D.paged_append(new, new, *pool.args[:2], *pool.args[2:], q_start=qs.cuda())
    for s in range(seqs):
        pages = [int(pool.table[s, j]) for j in range(-(-lens[s] // 16))]
        now, was = (torch.cat([x[p] for p in pages], 1)[:, :lens[s]] for x in (pool.k, before))
        if 0 < s < seqs - 2:
            assert (now[:, 30:] == 3).all() and torch.equal(now[:, :30], was[:, :30])
        else:
            assert torch.equal(now, was)


def test_beam_search_refuses_more_beams_than_a_reorder_takes():
    """batch x beams over 65 535 is refused before the encoder runs, not by the first step's reorder"""
    from fudanocr_amd.loss.transformer import Transformer as Characters
    from fudanocr_amd.loss.transformer_english_decomposition import Transformer as EnglishStrokes
    from fudanocr_amd.sld.model.transformer import Transformer as Strokes

    def never(*a, **kw):
        raise AssertionError("the encoder ran")
    for model, shape in ((Strokes("stroke"), (3, 32, 32)), (Characters(), (1, 32, 128)), (EnglishStrokes(), (4, 32, 128))):
        model.encoder.forward = never
        image = torch.zeros(1, *shape).expand(1024, *shape)
        _raises("65535", model.eval().beam_search, image, beams=64)
        _raises("65535", model.beam_search, torch.zeros(1, *shape).expand(65536, *shape), beams=1)
    _raises("65535", Strokes("stroke").eval().beam_search, None, beams=64, conv_feature=torch.zeros(1, 1, 1, 1).expand(1024, 1024, 8, 8))
