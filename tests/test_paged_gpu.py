"""The paged cache of keys and values (write, read back) and the attention over it, against plain forms in 64 bits."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

NAN = float("nan")


@pytest.fixture(params=["by size", "split", "chunk"])
def kernel(request):
    """The attention test that asks for it runs with the kernel the sizes choose and with each of the two."""
    import cudaop_b200 as ops
    assert ops.lib().b200q_paged_set_impl(["by size", "split", "chunk"].index(request.param)) == 0
    yield request.param
    ops.lib().b200q_paged_set_impl(0)


# ------------------------------------------------------------------------------------------------------ plain forms
def quantise_rows(x):
    """Per-row E4M3 by the library's rule, in the same 32-bit steps: (bytes, scales)."""
    x = x.float()
    a = x.abs().amax(-1)
    s = torch.where(a > 0, (a / 448.0).clamp(min=2.0 ** -126), torch.ones_like(a))
    q = (x * s.reciprocal().unsqueeze(-1)).to(torch.float8_e4m3fn).view(torch.uint8)
    bad = ~torch.isfinite(x).all(-1)
    return torch.where(bad.unsqueeze(-1), torch.zeros_like(q), q), torch.where(bad, torch.full_like(s, NAN), s)


def empty_cache(pages, heads, page, dim, fp8, garbage=True):
    """A cache whose every slot holds NaN, as memory that nobody wrote may."""
    shape = (pages, heads, page, dim)
    if fp8:
        fill = 0x7F if garbage else 0
        return [torch.full(shape, fill, dtype=torch.uint8, device="cuda"), torch.full(shape, fill, dtype=torch.uint8, device="cuda"),
                torch.full(shape[:3], NAN if garbage else 0.0, device="cuda"), torch.full(shape[:3], NAN if garbage else 0.0, device="cuda")]
    return [torch.full(shape, NAN if garbage else 0.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)] + [None, None]


def names(cache):
    return dict(zip(("k_cache", "v_cache", "k_scale", "v_scale"), cache))


class Batch:
    """Sequences of `kv` tokens whose last `n` are the new ones, in a cache with shuffled pages."""

    def __init__(self, n, kv, heads=8, kv_heads=2, dim=128, page=16, fp8=True, seed=0, spare=3, wide=2, cached=None):
        g = torch.Generator().manual_seed(seed + 131 * dim + page + fp8)
        self.n, self.kv, self.heads, self.kv_heads, self.dim, self.page, self.fp8 = n, kv, heads, kv_heads, dim, page, fp8
        cached = cached or [max(k, 0) for k in kv]
        need = [-(-c // page) for c in cached]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=g)
        self.table = torch.full((len(kv), max(need + [1]) + wide), -1, dtype=torch.int32)
        self.cache = empty_cache(self.pages, kv_heads, page, dim, fp8)
        self.k, self.v, at, slots = [], [], 0, []
        for b, c in enumerate(cached):
            self.table[b, :need[b]] = order[at:at + need[b]].int()
            at += need[b]
            j = torch.arange(c)
            slots.append(self.table[b][j // page].long() * page + j % page)
            self.k.append((torch.randn(c, kv_heads, dim, generator=g) * 1.5).bfloat16())
            self.v.append((torch.randn(c, kv_heads, dim, generator=g) * torch.exp(torch.randn(c, kv_heads, 1, generator=g))).bfloat16())
        import cudaop_b200 as ops
        if sum(cached):
            ops.paged_cache_write(torch.cat(self.k).cuda(), torch.cat(self.v).cuda(), torch.cat(slots).cuda(), **names(self.cache))
        self.q = torch.randn(sum(n), heads, dim, generator=g).bfloat16()
        self.cu = torch.tensor([0] + list(np.cumsum(n)), dtype=torch.int32)

    def held(self, b, name):
        """What the cache holds of sequence b, in 64 bits [tokens, kv_heads, dim]."""
        x = getattr(self, name)[b]
        if not self.fp8:
            return x.double()
        q, s = quantise_rows(x)
        return q.view(torch.float8_e4m3fn).double() * s.double().unsqueeze(-1)

    def call(self, q=None, **more):
        import cudaop_b200 as ops
        args = dict(page_table=self.table.cuda(), cu_q=self.cu.cuda(), kv_lens=torch.tensor(self.kv, dtype=torch.int32).cuda(),
                    max_q=max(self.n + [1]), return_lse=True, **names(self.cache))
        args.update(more)
        return ops.paged_attention((self.q if q is None else q).cuda(), **args)

    def expect(self, causal=True, window=0, scale=None, absent=()):
        """(out, lse, bound of out, bound of lse) in 64 bits.  absent: (sequence, page column) pairs that hold no tokens."""
        scale = self.dim ** -0.5 if scale is None else scale
        out, lse, tol, ltol = [], [], [], []
        group = self.heads // self.kv_heads
        for b, (n, kv) in enumerate(zip(self.n, self.kv)):
            q = self.q[int(self.cu[b]):int(self.cu[b]) + n].double()
            k, v = self.held(b, "k"), self.held(b, "v")
            kv_here = min(max(kv, 0), k.shape[0])
            k, v = k[:kv_here].repeat_interleave(group, 1), v[:kv_here].repeat_interleave(group, 1)
            p = torch.arange(n).unsqueeze(1) + (max(kv, 0) - n)
            j = torch.arange(kv_here).unsqueeze(0)
            seen = torch.ones(n, kv_here, dtype=torch.bool)
            if causal:
                seen &= j <= p
            if window:
                seen &= j > p - window
            for bb, col in absent:
                if bb == b:
                    seen &= (j // self.page != col)
            x = torch.einsum("nhd,khd->hnk", q, k) * scale
            mag = torch.einsum("nhd,khd->hnk", q.abs(), k.abs()) * abs(scale)
            x = torch.where(seen, x, torch.full_like(x, -math.inf))
            l = torch.logsumexp(x, 2) if kv_here else torch.full((self.heads, n), -math.inf, dtype=torch.float64)
            w = torch.where(seen, torch.exp(x - torch.where(l.isinf(), torch.zeros_like(l), l).unsqueeze(2)), torch.zeros_like(x))
            v0 = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
            o = torch.einsum("hnk,khd->nhd", w, v0)
            # a score: dim products added in 32 bits and two products with scales, relative to the sum of the magnitudes; the
            # maximum that is subtracted has the same error.  2^x: 2^-22, and its argument's rounding.
            worst = torch.where(seen, mag, torch.zeros_like(mag)).amax(2) if kv_here else torch.zeros(self.heads, n, dtype=torch.float64)
            delta = (worst * (self.dim + 8) * 2.0 ** -23 * 2 + 2.0 ** -20).t()
            # out: its own rounding; that of each p to bf16; the scores' errors
            share = torch.einsum("hnk,khd->nhd", w, v0.abs())
            out.append(o); lse.append(l.t())
            tol.append(2.0 ** -8 * o.abs() + (2.0 ** -8 + 2 * delta.unsqueeze(2)) * share + 1e-30)
            ltol.append(delta + 2.0 ** -21 * l.t().abs().nan_to_num(posinf=0.0))
        return torch.cat(out), torch.cat(lse), torch.cat(tol), torch.cat(ltol)

    def check(self, got, **how):
        import cudaop_b200 as ops
        torch.cuda.synchronize()
        assert ops.status() == 0
        out, lse = (t.double().cpu() for t in got)
        want, wlse, tol, ltol = self.expect(**how)
        T = want.shape[0]
        assert got[0].dtype == torch.bfloat16 and got[0].shape == self.q.shape and not out.isnan().any()
        err = (out[:T] - want).abs()
        assert (err <= tol).all(), f"out: {(err / tol).max():.3f} of the bound at {int((err / tol).argmax())}"
        none = wlse == -math.inf
        assert torch.equal(none, lse[:T] == -math.inf)
        assert (out[:T][none] == 0).all()
        err = (lse[:T] - wlse).abs()[~none]
        assert (err <= ltol[~none]).all(), f"lse: {(err / ltol[~none]).max():.3f} of the bound"


# ------------------------------------------------------------------------------------------------------ write and read
@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens,heads,page", [(1, 1, 16), (7, 3, 32), (33, 8, 64), (500, 5, 128), (1000, 2, 16)])
def test_write_is_exact_and_touches_nothing_else(tokens, heads, page, dim, fp8):
    import cudaop_b200 as ops
    g = torch.Generator().manual_seed(tokens + dim)
    pages = tokens // page + 3
    cache = empty_cache(pages, heads, page, dim, fp8)
    before = [None if t is None else t.clone() for t in cache]
    qkv = (torch.randn(tokens, 3 * heads * dim + 8, generator=g) * torch.exp2(torch.randint(-30, 30, (tokens, 1), generator=g).float())).bfloat16()
    qkv[0] = 0                                                       # a row of zeros
    if tokens > 6:
        qkv[5, heads * dim] = 2.0 ** -133                            # a row whose largest value is next to it: stays finite
    wide = qkv.cuda()
    k = wide[:, heads * dim:2 * heads * dim].unflatten(1, (heads, dim))
    v = wide[:, 2 * heads * dim:3 * heads * dim].unflatten(1, (heads, dim))
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[tokens // 2:][::4] = -1
    if tokens > 6:
        slots[3], slots[4], slots[6] = pages * page, 2 ** 40, -2 ** 40       # behind the cache
    ops.paged_cache_write(k, v, slots.cuda(), **names(cache))
    torch.cuda.synchronize()
    fine = (slots >= 0) & (slots < pages * page)
    at = slots[fine]
    for i, x in enumerate((k, v)):
        x = x.cpu()[fine]
        want, got = before[i].cpu(), cache[i].cpu()
        if fp8:
            q, s = quantise_rows(x)
            scales = before[2 + i].cpu()
            scales[at // page, :, at % page] = s
            assert np.array_equal(scales.numpy().view(np.uint32), cache[2 + i].cpu().numpy().view(np.uint32))
            want[at // page, :, at % page] = q
            assert torch.equal(want, got)
        else:
            want[at // page, :, at % page] = x
            assert torch.equal(want.view(torch.int16), got.view(torch.int16))


def test_write_of_rows_that_are_not_finite():
    import cudaop_b200 as ops
    cache = empty_cache(2, 2, 16, 64, True, garbage=False)
    k = torch.ones(4, 2, 64, dtype=torch.bfloat16)
    v = k.clone()
    k[0, 0, 5], k[1, 1, 63], v[2, 0, 0], v[3, 1, 9] = NAN, math.inf, -math.inf, -NAN
    ops.paged_cache_write(k.cuda(), v.cuda(), torch.tensor([0, 1, 17, 31]).cuda(), **names(cache))
    back = ops.paged_cache_read(page_table=torch.tensor([[0, 1]], dtype=torch.int32).cuda(), cu_kv=torch.tensor([0, 32], dtype=torch.int32).cuda(),
                                total=32, **names(cache))
    kb, vb = (t.cpu().float() for t in back)
    want_k = torch.zeros(32, 2, 64); want_v = torch.zeros(32, 2, 64)
    for t, s in enumerate([0, 1, 17, 31]):
        want_k[s], want_v[s] = 1, 1
    want_k[0, 0], want_k[1, 1], want_v[17, 0], want_v[31, 1] = NAN, NAN, NAN, NAN
    assert torch.equal(kb.isnan(), want_k.isnan()) and torch.equal(vb.isnan(), want_v.isnan())
    assert torch.equal(kb.nan_to_num(7.0), want_k.nan_to_num(7.0)) and torch.equal(vb.nan_to_num(7.0), want_v.nan_to_num(7.0))
    assert not (cache[0] == 0x7F).any() and not (cache[1] == 0xFF).any()


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("dim,page,kv_heads", [(64, 16, 3), (128, 64, 2), (128, 128, 1), (64, 32, 8)])
def test_read_back(dim, page, kv_heads, fp8):
    import cudaop_b200 as ops
    kv = [1, 0, 200, 16, 129, 77]
    b = Batch([0] * len(kv), kv, heads=kv_heads, kv_heads=kv_heads, dim=dim, page=page, fp8=fp8)
    b.table[2, 1] = b.pages                                          # not in the cache
    b.table[4, 0] = -5
    total = sum(kv) + 9
    cu = torch.tensor([0] + list(np.cumsum(kv)), dtype=torch.int32)
    want = []
    for name in ("k", "v"):
        rows = []
        for s, n in enumerate(kv):
            x = b.held(s, name).float().bfloat16() if not fp8 else None
            if fp8:
                q, sc = quantise_rows(getattr(b, name)[s])
                x = (q.view(torch.float8_e4m3fn).float() * sc.unsqueeze(-1)).bfloat16()
            if s == 2:
                x[page:2 * page] = 0
            if s == 4:
                x[:page] = 0
            rows.append(x)
        want.append(torch.cat(rows + [torch.zeros(9, kv_heads, dim, dtype=torch.bfloat16)]))
    got = ops.paged_cache_read(page_table=b.table.cuda(), cu_kv=cu.cuda(), total=total, **names(b.cache))
    for x, y in zip(got, want):
        assert torch.equal(x.cpu().float(), y.float())
    # rows behind the last sequence stay as they are in tensors that are given
    given = [torch.full((total, kv_heads, dim), 5.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    got = ops.paged_cache_read(page_table=b.table.cuda(), cu_kv=cu.cuda(), total=total, k_out=given[0], v_out=given[1], **names(b.cache))
    for x, y, z in zip(got, want, given):
        assert x.data_ptr() == z.data_ptr()
        assert torch.equal(x[:sum(kv)].cpu().float(), y[:sum(kv)].float()) and (x[sum(kv):] == 5.0).all()


@pytest.mark.parametrize("start", [-1, -40, -2 ** 31 + 5, -2 ** 31])
def test_read_back_with_starts_below_zero(start):
    """A first start below zero counts as zero, as in the attention: the tokens are those from the first one on."""
    import cudaop_b200 as ops
    b = Batch([0, 0], [70, 30], heads=2, kv_heads=2, dim=64, page=16, fp8=True)
    args = dict(page_table=b.table.cuda(), total=100, **names(b.cache))
    want = ops.paged_cache_read(cu_kv=torch.tensor([0, 70, 100], dtype=torch.int32).cuda(), **args)
    got = ops.paged_cache_read(cu_kv=torch.tensor([start, 70, 100], dtype=torch.int32).cuda(), **args)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ------------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (8, 1), (12, 2), (32, 4), (40, 2)])
def test_one_token(kernel, heads, kv_heads, dim, fp8):
    """Decode: lengths from one token to many tiles, at and around the borders of pages and tiles."""
    kv = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500, 1000, 3]
    b = Batch([1] * len(kv), kv, heads, kv_heads, dim, page=16, fp8=fp8)
    b.check(b.call())


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dim,fp8", [(128, True), (64, True), (128, False), (64, False)])
def test_page_sizes_and_mixed_chunks(kernel, dim, fp8, page):
    n = [1, 5, 0, 33, 2, 130, 64]
    kv = [300, 5, 40, 200, 1000, 131, 64]
    b = Batch(n, kv, 8, 2, dim, page, fp8)
    b.check(b.call())


@pytest.mark.parametrize("dim,fp8", [(128, True), (64, False)])
@pytest.mark.parametrize("window", [1, 2, 16, 100, 5000])
def test_windows(kernel, window, dim, fp8):
    b = Batch([1, 7, 100, 20, 300], [900, 7, 400, 21, 700], 8, 2, dim, 16, fp8)
    b.check(b.call(window=window), window=window)


@pytest.mark.parametrize("dim,fp8", [(64, True), (128, False), (128, True)])
def test_every_key_is_seen_without_causal(kernel, dim, fp8):
    b = Batch([1, 7, 100, 300], [900, 7, 400, 700], 8, 4, dim, 32, fp8)
    b.check(b.call(causal=False), causal=False)


@pytest.mark.parametrize("dim,fp8", [(128, True), (128, False), (64, True)])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_that_see_nothing(kernel, causal, dim, fp8):
    """Fewer cached tokens than new ones, none at all, a negative length: zero rows and lse -inf."""
    b = Batch([4, 3, 1, 40, 2, 300], [2, 0, 0, 7, -3, 290], 8, 2, dim, 16, fp8)
    b.check(b.call(causal=causal), causal=causal)


@pytest.mark.parametrize("dim,fp8", [(128, True), (64, False)])
@pytest.mark.parametrize("n", [1, 140])
def test_pages_that_are_not_in_the_cache_are_left_out(kernel, n, dim, fp8):
    b = Batch([n, n], [400, 150], 8, 2, dim, 16, fp8)
    absent = [(0, 0), (0, 7), (0, 24), (1, 3)]
    for i, (s, col) in enumerate(absent):
        b.table[s, col] = [-1, b.pages, 2 ** 31 - 1, -2 ** 31][i]
    b.check(b.call(), absent=absent)
    for col in range(10):                                            # ... and a sequence none of whose pages are
        b.table[1, col] = -1
    b.check(b.call(), absent=absent[:3] + [(1, col) for col in range(10)])


def test_length_longer_than_the_table(kernel):
    """Keys behind the table's last page are not there; positions still count from kv_lens."""
    b = Batch([3], [100], 4, 2, 128, 16, True, wide=0)
    b.kv = [130]                                                     # 7 pages hold 112 slots; 100 are written, the rest is NaN
    b.table[0, 6] = -1
    b.check(b.call(), absent=[(0, 6)])


@pytest.mark.parametrize("n", [1, 9, 200])
def test_strided_queries_scale_and_given_output(kernel, n):
    """Queries inside a fused projection's output; rows of no sequence stay as they are in a given output, else are zero."""
    b = Batch([n, 2 * n], [300, 450], 8, 2, 128, 64, True)
    T = 3 * n
    wide = torch.full((T + 5, 12 * 128 + 16), NAN, dtype=torch.bfloat16)
    wide[:T, 16:16 + 8 * 128] = b.q.flatten(1)
    q = wide.cuda()[:, 16:16 + 8 * 128].unflatten(1, (8, 128))
    out, lse = b.call(q=q, scale=0.25)
    assert (out[T:] == 0).all() and (lse[T:] == -math.inf).all()
    b.check((out[:T], lse[:T]), scale=0.25)
    given = torch.full((T + 5, 8, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    out2, _ = b.call(q=q, scale=0.25, out=given)
    assert out2.data_ptr() == given.data_ptr() and (given[T:] == 3.0).all() and torch.equal(given[:T], out[:T])
    # heads first in memory
    q = b.q.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    b.check(b.call(q=q))


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-3])
def test_scales_that_are_negative_zero_and_small(kernel, scale, fp8):
    b = Batch([1, 30, 150], [200, 64, 150], 8, 2, 64, 16, fp8)
    b.check(b.call(scale=scale), scale=scale)


@pytest.mark.parametrize("fp8", [True, False])
def test_groups_larger_than_a_block_of_rows(kernel, fp8):
    b = Batch([1, 3, 2], [100, 3, 257], 300, 1, 64, 32, fp8)
    b.check(b.call())


@pytest.mark.parametrize("dim,fp8", [(128, True), (64, False)])
def test_queries_of_very_different_size(kernel, dim, fp8):
    """Elements of a row, and rows, from 2^-60 to 2^40: an E4M3 cache's fp16 queries are scaled row by row."""
    b = Batch([40], [300], 4, 1, dim, 16, fp8)
    g = torch.Generator().manual_seed(8)
    q = b.q.float() * torch.exp2(torch.randint(-12, 1, b.q.shape, generator=g).float())
    q[::5] *= 2.0 ** -60
    q[1::5] *= 2.0 ** 20                                             # (these rows' scores pick one key each)
    b.q = q.bfloat16()
    b.check(b.call())


def test_lengths_that_contradict_the_tensors_stay_inside_them(kernel):
    """Starts that go back, pass the end or are negative, lengths beyond the table: rows of such a call are not defined,
    but nothing is read or written outside the tensors."""
    b = Batch([20, 20, 20], [100, 100, 100], 4, 2, 64, 16, True)
    for cu in ([0, 50, 10, 60], [-5, 10, 1000, 2000], [70, 80, 90, 100], [60, 0, 0, 0], [-2 ** 31, 2 ** 31 - 1, 0, 7]):
        for kv in ([100, 100, 100], [2 ** 31 - 1, -2 ** 31, 5]):
            guard = torch.full((60 + 64, 4, 64), 9.0, dtype=torch.bfloat16, device="cuda")
            b.call(cu_q=torch.tensor(cu, dtype=torch.int32).cuda(), kv_lens=torch.tensor(kv, dtype=torch.int32).cuda(), out=guard[32:92])
            torch.cuda.synchronize()
            assert (guard[:32] == 9.0).all() and (guard[92:] == 9.0).all()
    import cudaop_b200 as ops
    assert ops.status() == 0
    b.check(b.call())


def test_overlapping_chunks_beyond_the_count_of_tiles_do_nothing(kernel):
    """4096 sequences that all claim the same 20000 rows and a table of 10^6 tokens: more tiles than 32 bits count."""
    import cudaop_b200 as ops
    seqs, T = 4096, 20000
    cu = torch.zeros(seqs + 1, dtype=torch.int32)
    cu[1::2] = T
    cache = names(empty_cache(4, 1, 128, 64, True))
    out = torch.full((T, 8, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    table = torch.full((seqs, 8192), -1, dtype=torch.int32, device="cuda")
    ops.paged_attention(torch.zeros_like(out), page_table=table, cu_q=cu.cuda(), kv_lens=torch.full((seqs,), 2 ** 20, dtype=torch.int32).cuda(),
                        max_q=T, causal=False, out=out, **cache)
    torch.cuda.synchronize()
    assert ops.status() == 0 and (out == 9.0).all()


@pytest.mark.parametrize("n,fp8", [(1, True), (1, False), (40, True), (200, False)])
def test_large_scores_and_equal_runs(kernel, n, fp8):
    """Scores of hundreds: the running maximum moves at every tile; and two runs give the same bits."""
    b = Batch([n, n], [1000, 777], 16, 2, 128, 32, fp8, seed=5)
    b.q = (b.q.float() * 20).bfloat16()
    got = b.call()
    b.check(got)
    again = b.call()
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_a_nan_key_reaches_the_rows_that_see_it(kernel):
    """E4M3 rows with NaN: rows that see the token are NaN, rows in front of it are as if it were not there."""
    import cudaop_b200 as ops
    b = Batch([8], [64], 2, 1, 128, 16, True)
    bad = b.v[0][60:61].clone()
    bad[0, 0, 3] = NAN
    slot = int(b.table[0, 60 // 16]) * 16 + 60 % 16
    ops.paged_cache_write(b.k[0][60:61].cuda(), bad.cuda(), torch.tensor([slot]).cuda(), **names(b.cache))
    out, lse = b.call()
    assert out[4:].isnan().all()                                     # positions 60 .. 63
    want, wlse, tol, ltol = b.expect()
    assert ((out[:4].double().cpu() - want[:4]).abs() <= tol[:4]).all()


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("n,group,dim", [(8, 2, 128), (150, 4, 64), (30, 8, 128)])
def test_values_that_are_not_finite_reach_the_rows_that_see_them_alone(kernel, n, group, dim, window):
    """bf16 cache: NaN and infinities in values (and keys) of tokens that some rows see and others do not."""
    import cudaop_b200 as ops
    kv = 200
    b = Batch([n], [kv], 2 * group, 2, dim, 16, False, seed=7)
    g = torch.Generator().manual_seed(n)
    odd = {kv - 1: NAN, kv - n // 2: math.inf, kv - n: -math.inf, kv - n + 1: math.inf, 100: NAN, 3: -math.inf}
    for j, value in odd.items():
        b.v[0][j, torch.randint(0, 2, (1,), generator=g), torch.randint(0, dim, (3,), generator=g)] = value
    b.v[0][kv - n + 2, 1] = NAN                                      # a whole row
    at = torch.arange(kv)
    slots = b.table[0][at // 16].long() * 16 + at % 16
    ops.paged_cache_write(b.k[0].cuda(), b.v[0].cuda(), slots.cuda(), **names(b.cache))
    out, lse = b.call(window=window)
    torch.cuda.synchronize()
    assert ops.status() == 0
    want, wlse, tol, ltol = b.expect(window=window)
    # what the rows that see a value that is not finite have in its column
    v = b.v[0].double().repeat_interleave(group, 1)
    bad = torch.where(torch.isfinite(v), torch.zeros_like(v), v)
    p, j = torch.arange(n).unsqueeze(1) + kv - n, torch.arange(kv).unsqueeze(0)
    seen = (j <= p) & ((j > p - window) if window else True)
    for i in range(n):
        want[i] += bad[seen[i]].sum(0)
    out, lse = out.double().cpu(), lse.double().cpu()
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out.isinf(), want.isinf()) and torch.equal(out[want.isinf()], want[want.isinf()])
    fine = torch.isfinite(want)
    assert fine.float().mean() > 0.3 and not fine.all()
    assert ((out - want).abs()[fine] <= tol[fine]).all()
    assert ((lse - wlse).abs() <= ltol).all()


def test_many_sequences_and_a_chunk_bound_that_is_too_small(kernel):
    g = np.random.default_rng(3)
    kv = [int(x) for x in g.integers(1, 90, 700)]
    b = Batch([1] * 700, kv, 4, 2, 64, 16, True)
    b.check(b.call())
    b = Batch([3, 50, 260], [30, 50, 300], 8, 2, 128, 16, True)
    b.check(b.call(max_q=1))
    b.check(b.call(max_q=10 ** 6))


def test_offsets_that_pass_32_bits(kernel):
    """A cache of more than 2^32 elements, its tokens at both ends."""
    import cudaop_b200 as ops
    pages, heads, page, dim = 280000, 8, 16, 128
    assert pages * heads * page * dim > 2 ** 32
    k_cache = torch.empty((pages, heads, page, dim), dtype=torch.uint8, device="cuda")
    v_cache = torch.empty_like(k_cache)
    scales = [torch.empty((pages, heads, page), device="cuda") for _ in range(2)]
    small = Batch([1, 20], [40, 70], 8, heads, dim, page, True)
    table = small.table.clone()
    for old in range(small.pages):
        table[small.table == old] = pages - 1 - old * 37 if old % 2 else old
    slots = torch.cat([table[b][torch.arange(c) // page].long() * page + torch.arange(c) % page for b, c in enumerate(small.kv)])
    ops.paged_cache_write(torch.cat(small.k).cuda(), torch.cat(small.v).cuda(), slots.cuda(), k_cache, v_cache, *scales)
    small.table, small.cache = table, [k_cache, v_cache] + scales
    small.check(small.call())
    cu = torch.tensor([0, 40, 110], dtype=torch.int32)
    kb, _ = ops.paged_cache_read(page_table=table.cuda(), cu_kv=cu.cuda(), total=110, **names(small.cache))
    q, s = quantise_rows(torch.cat(small.k))
    assert torch.equal(kb.cpu(), (q.view(torch.float8_e4m3fn).float() * s.unsqueeze(-1)).bfloat16())


@pytest.mark.parametrize("n", [1, 150])
def test_side_stream_and_graph(n):
    """On another stream; captured once and replayed with other lengths and pages; two graphs in flight at once."""
    b = Batch([n, n], [600, 333], 8, 2, 128, 16, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = b.call()
    side.synchronize()
    b.check(got)
    c = Batch([n, n], [200, 599], 8, 2, 128, 16, True, seed=1)
    import cudaop_b200 as ops
    graphs = []
    for x in (b, c):
        static = dict(page_table=x.table.cuda(), cu_q=x.cu.cuda(), kv_lens=torch.tensor(x.kv, dtype=torch.int32).cuda(), **names(x.cache))
        q = x.q.cuda()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            held = ops.paged_attention(q, max_q=n, return_lse=True, **static)
        graphs.append((graph, held, {**static, "q": q}))           # a replay reads what the capture read
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for (graph, _, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for x, (_, held, _) in zip((b, c), graphs):
        x.check(held)
    b.kv = [150, 333 - 12]
    graphs[0][2]["kv_lens"].copy_(torch.tensor(b.kv))
    graphs[0][0].replay()
    b.check(graphs[0][1])


@pytest.mark.parametrize("n", [1, 150])
def test_after_work_that_is_still_running(n):
    """The cache write, the attention and what reads it in one stream, behind a kernel that takes long."""
    import cudaop_b200 as ops
    b = Batch([n, n], [600, 333], 8, 2, 128, 16, True)
    want = b.call()
    big = torch.empty(1 << 28, device="cuda")
    fresh = names(empty_cache(b.pages, 2, 16, 128, True))
    slots = torch.cat([b.table[s][torch.arange(c) // 16].long() * 16 + torch.arange(c) % 16 for s, c in enumerate(b.kv)]).cuda()
    k, v = torch.cat(b.k).cuda(), torch.cat(b.v).cuda()
    args = dict(page_table=b.table.cuda(), cu_q=b.cu.cuda(), kv_lens=torch.tensor(b.kv, dtype=torch.int32).cuda(), max_q=n, return_lse=True)
    q = b.q.cuda()
    torch.cuda.synchronize()
    for _ in range(3):
        big.normal_()
        ops.paged_cache_write(k, v, slots, **fresh)
        got = ops.paged_attention(q, **args, **fresh)
        copy = got[0].clone()
        for t in fresh.values():
            t.view(torch.uint8).fill_(0x7F)
        assert torch.equal(copy, want[0]) and torch.equal(got[1], want[1])


def test_a_layer_of_quantised_inference():
    """The operators together, as a decoder layer uses them: quantise, project to q, k, v (MXFP4), write the new tokens'
    keys and values, attend to the cache, quantise, project back.  Prefill in two chunks, then single tokens."""
    import cudaop_b200 as ops
    heads, kv_heads, dim, hidden, page = 8, 2, 64, 512, 16
    g = torch.Generator().manual_seed(11)
    wqkv = ops.quant_rows_mxfp4((torch.randn((heads + 2 * kv_heads) * dim, hidden, generator=g) / hidden ** 0.5).bfloat16().cuda())
    wo = ops.quant_rows_mxfp4((torch.randn(hidden, heads * dim, generator=g) / hidden ** 0.5).bfloat16().cuda())
    lens = [100, 37]
    x = torch.randn(sum(lens), hidden, generator=g).bfloat16().cuda()
    first = [0, 100]
    pages = 20
    cache = names(empty_cache(pages, kv_heads, page, dim, True))
    table = torch.randperm(pages, generator=g).int().view(2, 10)

    def step(done, upto):
        """Tokens done[b] .. upto[b] of each sequence through the layer."""
        rows = torch.cat([torch.arange(first[b] + done[b], first[b] + upto[b]) for b in range(2)])
        slots = torch.cat([table[b][torch.arange(done[b], upto[b]) // page].long() * page + torch.arange(done[b], upto[b]) % page for b in range(2)])
        xq, xs = ops.quant_rows_mxfp4(x[rows.cuda()])
        qkv = ops.gemm_mxfp4(xq, xs, *wqkv, blocked=True)
        q, k, v = qkv.unflatten(1, (-1, dim)).split([heads, kv_heads, kv_heads], 1)
        ops.paged_cache_write(k, v, slots.cuda(), **cache)
        n = [u - d for d, u in zip(done, upto)]
        o = ops.paged_attention(q, page_table=table.cuda(), cu_q=torch.tensor([0, n[0], n[0] + n[1]], dtype=torch.int32).cuda(),
                                kv_lens=torch.tensor(upto, dtype=torch.int32).cuda(), max_q=max(n), **cache)
        oq, os_ = ops.quant_rows_mxfp4(o.flatten(1))
        return rows, qkv, o, ops.gemm_mxfp4(oq, os_, *wo, blocked=True)

    qkv = torch.zeros(sum(lens), (heads + 2 * kv_heads) * dim, dtype=torch.bfloat16)
    o = torch.zeros(sum(lens), heads, dim, dtype=torch.bfloat16)
    y = torch.zeros(sum(lens), hidden, dtype=torch.bfloat16)
    done = [0, 0]
    for upto in ([60, 20], [98, 35], [99, 36], [100, 37]):
        rows, a, b, c = step(done, upto)
        qkv[rows], o[rows], y[rows] = a.cpu(), b.cpu(), c.cpu()
        done = upto
    torch.cuda.synchronize()
    assert ops.status() == 0
    # the same from the whole sequences at once, every operator's 64-bit form applied to what the one before gave
    for b in range(2):
        part = qkv[first[b]:first[b] + lens[b]].unflatten(1, (-1, dim))
        ref = Batch([lens[b]], [lens[b]], heads, kv_heads, dim, page, True)
        ref.q, ref.k[0], ref.v[0] = part[:, :heads], part[:, heads:heads + kv_heads], part[:, heads + kv_heads:]
        want, _, tol, _ = ref.expect()
        err = (o[first[b]:first[b] + lens[b]].double() - want).abs()
        assert (err <= tol).all()
    oq, os_ = ops.quant_rows_mxfp4(o.flatten(1).cuda())
    whole = ops.gemm_mxfp4(oq, os_, *wo, blocked=True).cpu()
    # the rows' products do not depend on the batch they were computed in, up to the order of 32-bit sums before one rounding
    assert ((whole.double() - y.double()).abs() <= 2.0 ** -7 * whole.double().abs() + 2.0 ** -12).all()


# ------------------------------------------------------------------------------------------------------ value scales of an E4M3 cache
class Scaled(Batch):
    """A batch whose value scales are given, not those that the write computes: vs[b] is [tokens, kv_heads]."""

    def __init__(self, vs, n, kv, **how):
        super().__init__(n, kv, fp8=True, **how)
        self.vs = [s.float() for s in vs]
        for b, s in enumerate(self.vs):
            at = torch.arange(s.shape[0])
            slot = self.table[b][at // self.page].long() * self.page + at % self.page
            self.cache[3][slot.cuda() // self.page, :, slot.cuda() % self.page] = s.cuda()

    def held(self, b, name):
        if name == "k":
            return super().held(b, name)
        q, _ = quantise_rows(self.v[b])
        return q.view(torch.float8_e4m3fn).double() * self.vs[b].double().unsqueeze(-1)


@pytest.mark.parametrize("dim,page", [(128, 64), (64, 16)])
@pytest.mark.parametrize("n", [1, 30, 150])
@pytest.mark.parametrize("s", [0.0, 2.0 ** -126, 2.0 ** -113, 2.0 ** -105])
@pytest.mark.parametrize("behind", [0, 200])
def test_value_scales_that_are_zero_or_tiny(kernel, behind, s, n, dim, page):
    """A cache of zeros read before every slot is written, one quantised elsewhere, rows next to zero: whole tiles of such scales,
    alone and with tiles of ordinary ones behind them."""
    kv = [300, 160]
    vs = [torch.cat([torch.full((k, 2), s), torch.rand(behind, 2, generator=torch.Generator().manual_seed(k)) + 0.01]) for k in kv]
    b = Scaled(vs, [n, n], [k + behind for k in kv], heads=8, kv_heads=2, dim=dim, page=page)
    got = b.call()
    torch.cuda.synchronize()
    assert torch.isfinite(got[0]).all()
    out, lse = got
    want, wlse, tol, ltol = b.expect()
    # p * scale may round to zero where it is far below 2^-63: half a step of fp16 (2^-25) of at least 2^-74, for each key, times 448
    tol = tol + 500 * 448 * 2.0 ** -99
    assert ((out.double().cpu() - want).abs() <= tol).all()
    assert ((lse.double().cpu() - wlse).abs() <= ltol).all()


def shares(b, causal=True, window=0):
    """Per sequence, from the definition in 64 bits: the weights [heads, n, keys] of the softmax."""
    group = b.heads // b.kv_heads
    for s, (n, kv) in enumerate(zip(b.n, b.kv)):
        q, k = b.q[int(b.cu[s]):int(b.cu[s]) + n].double(), b.held(s, "k").repeat_interleave(group, 1)
        p, j = torch.arange(n).unsqueeze(1) + kv - n, torch.arange(kv).unsqueeze(0)
        seen = (j <= p) | (not causal)
        if window:
            seen &= j > p - window
        x = torch.einsum("nhd,khd->hnk", q, k) * b.dim ** -0.5
        yield s, torch.softmax(torch.where(seen, x, torch.full_like(x, -math.inf)), 2)


def check_scaled(b, **how):
    """Against 64 bits, with a bound made of what each row itself uses: the share of p |v| that it sees, and the loss of fp16."""
    import cudaop_b200 as ops
    out, lse = b.call(**how)
    torch.cuda.synchronize()
    assert ops.status() == 0
    want, wlse, tol, ltol = b.expect(**how)
    # p * scale is held in fp16 times 2^11 / 2^n: half a step of its small numbers, 2^-25, is 2^-36 2^n for each key; 2^n is at most
    # 2^13 times the largest p * scale that the row sees (2^12 of spread, and up to 2 from the scale to the power of two above it).
    # The tensor-core kernel may hold a first part on a base that is 2^4 below.
    extra = []
    for s, w in shares(b, **how):
        vs = b.vs[s].double().repeat_interleave(b.heads // b.kv_heads, 1)
        top = (w * vs.t().unsqueeze(1)).amax(2)                      # [heads, n]
        codes = quantise_rows(b.v[s])[0].view(torch.float8_e4m3fn).double().abs().sum(0).repeat_interleave(b.heads // b.kv_heads, 0)
        extra.append(2.0 ** -23 * top.t().unsqueeze(2) * codes)
    tol = (tol - 1e-30) + torch.cat(extra) + 2.0 ** -133             # (... and half a step of bf16's smallest numbers)
    err = (out.double().cpu() - want).abs()
    assert (err <= tol).all(), f"out: {(err / tol).max():.3f} of the bound"
    assert ((lse.double().cpu() - wlse).abs() <= ltol).all()


@pytest.mark.parametrize("dim,page", [(128, 64), (64, 16)])
@pytest.mark.parametrize("n", [1, 30, 150])
@pytest.mark.parametrize("s", [2.0 ** -126, 2.0 ** -113, 2.0 ** -70, 2.0 ** 100])
def test_value_scales_far_from_one_keep_their_bits(kernel, s, n, dim, page):
    """All scales near the same power of two: relative errors are those of ordinary ones."""
    g = torch.Generator().manual_seed(n)
    check_scaled(Scaled([s * (1 + torch.rand(k, 2, generator=g)) for k in (300, 160)], [n, n], [300, 160], heads=8, kv_heads=2, dim=dim, page=page))


@pytest.mark.parametrize("dim,page", [(128, 64), (64, 16)])
@pytest.mark.parametrize("n", [1, 30, 150])
@pytest.mark.parametrize("how", ["keys", "tiles", "tiles, down", "zeros between"])
def test_value_scales_of_wide_spread(kernel, how, n, dim, page):
    """Scales from 2^-40 to 2^40 key by key, and from 2^-126 to 2^60 and back tile by tile."""
    g = torch.Generator().manual_seed(n)
    kv = [600, 400]
    vs = []
    for k in kv:
        if how == "keys":
            s = torch.exp2(torch.randint(-40, 41, (k, 2), generator=g).float())
        elif how == "zeros between":
            s = torch.rand(k, 2, generator=g) * (torch.rand(k, 2, generator=g) < 0.5)
        else:
            e = torch.tensor([-126.0, 0.0, 60.0, -50.0, 3.0])[torch.arange(k) // 128]
            s = torch.exp2(e.flip(0) if how == "tiles, down" else e).unsqueeze(1).repeat(1, 2)
        vs.append(s)
    check_scaled(Scaled(vs, [n, n], kv, heads=8, kv_heads=2, dim=dim, page=page))


@pytest.mark.parametrize("dim,page", [(128, 64), (64, 16)])
@pytest.mark.parametrize("n,window", [(8, 0), (8, 40), (150, 0), (150, 100), (300, 130)])
@pytest.mark.parametrize("up", [45, 100])
def test_a_huge_value_reaches_the_rows_that_see_it_alone(kernel, up, n, window, dim, page):
    """One finite token whose value scale is 2^45 (2^100) times the others': rows in front of it, and rows whose window it has
    left, are as exact as without it; so are rows that give it next to no weight."""
    kv = 400
    vs = torch.rand(kv, 2, generator=torch.Generator().manual_seed(n)) + 0.5
    vs[kv - n // 2, 0] *= 2.0 ** up                                  # new itself: hidden from the first half of the rows
    vs[kv - n - 5, 1] *= 2.0 ** up                                   # with a window of 100 or 130: seen by the first rows only
    check_scaled(Scaled([vs], [n], [kv], heads=8, kv_heads=2, dim=dim, page=page), window=window)


@pytest.mark.parametrize("dim,page", [(128, 64), (64, 16)])
@pytest.mark.parametrize("n", [1, 30, 150])
def test_a_huge_value_of_next_to_no_weight(kernel, n, dim, page):
    import cudaop_b200 as ops
    kv, at = 400, 200
    vs = torch.rand(kv, 2, generator=torch.Generator().manual_seed(n)) + 0.5
    vs[at] *= 2.0 ** 45
    b = Scaled([vs], [n], [kv], heads=8, kv_heads=2, dim=dim, page=page)
    b.q = b.q.abs()
    b.k[0][at] = -64.0 * dim ** -0.5                                 # scores near -50 for every row: a weight near 2^-75, times 2^45
    slot = int(b.table[0, at // page]) * page + at % page
    ops.paged_cache_write(b.k[0][at:at + 1].cuda(), b.v[0][at:at + 1].cuda(), torch.tensor([slot]).cuda(), **names(b.cache))
    b.cache[3][slot // page, :, slot % page] = vs[at].cuda()
    check_scaled(b)


def test_a_nan_scale_of_a_key_reaches_the_rows_that_see_it(kernel):
    """NaN in a key's scale: rows that see the token are NaN, lse included, rows in front of it as if it were not there."""
    for n, at in ((8, 60), (150, 100)):
        b = Batch([n], [at + 4 if n == 8 else 170], 4, 1, 128, 16, True)
        kv = b.kv[0]
        b.cache[2][int(b.table[0, at // 16]), :, at % 16] = NAN
        out, lse = b.call()
        front = at - (kv - n)
        assert out[front:].isnan().all() and lse[front:].isnan().all()
        want, wlse, tol, ltol = b.expect()
        assert ((out[:front].double().cpu() - want[:front]).abs() <= tol[:front]).all()
        assert ((lse[:front].double().cpu() - wlse[:front]).abs() <= ltol[:front]).all()


@pytest.mark.parametrize("dim,fp8", [(128, True), (64, True), (128, False)])
@pytest.mark.parametrize("scale", [1e-6, 1e-8, -1e-12, 1e-30, 1e-38])
def test_rows_of_zeros_and_next_to_zero_with_a_small_scale(kernel, scale, dim, fp8):
    """The power of two of a row times the softmax scale may leave the range of the numbers: all visible keys count alike."""
    b = Batch([30, 150], [64, 300], 8, 2, dim, 16, fp8)
    b.q[::3] = 0
    b.q[1::3] = (b.q[1::3].float() * 2.0 ** -120).bfloat16()
    b.check(b.call(scale=scale), scale=scale)


@pytest.mark.parametrize("dim,fp8", [(128, True), (64, False)])
@pytest.mark.parametrize("window", [2 ** 30, 2 ** 31 - 1, 2 ** 62])
def test_windows_that_hide_nothing(kernel, window, dim, fp8):
    """The largest windows, with chunks that are longer than what is cached (their first positions are negative)."""
    import cudaop_b200 as ops
    b = Batch([40, 3, 300], [7, 100, 290], 8, 2, dim, 16, fp8)
    want = b.call()
    got = b.call(window=window)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    if window < 2 ** 31:                                             # ... and through the C ABI
        L = ops.lib()
        q, table, cu, lens = b.q.cuda(), b.table.cuda(), b.cu.cuda(), torch.tensor(b.kv, dtype=torch.int32).cuda()
        out = torch.zeros_like(q)
        ws = torch.empty(L.b200q_paged_attention_workspace_bytes(dim), dtype=torch.uint8, device="cuda")
        at = [t if t is None else t.data_ptr() for t in (q, *b.cache, table, cu, lens, out, None)]
        assert L.b200q_paged_attention(*at, 3, q.shape[0], 8, 2, dim, q.stride(0), q.stride(1), 300, table.shape[1], b.pages, 16, fp8,
                                       dim ** -0.5, 1, window, 1, ws.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out, want[0])


# ------------------------------------------------------------------------------------------------------ bits of the probabilities
@pytest.mark.parametrize("n", [1, 20])
@pytest.mark.parametrize("dim,fp8", [(128, True), (64, True), (128, False), (64, False)])
def test_bits_of_the_probabilities(kernel, dim, fp8, n):
    """Two kinds of keys, half of them with p = 1 and half with a p that differs by row, and values of opposite sign that nearly cancel
    in some columns: there the rounding of the output is small, and that of p shows undiluted, since all its errors agree."""
    import cudaop_b200 as ops
    kv, heads, scale = 200, 16, 0.25
    b = Batch([n], [kv], heads, 1, dim, 16, fp8, seed=2)
    g = torch.Generator().manual_seed(n)
    b.q = torch.zeros(n, heads, dim, dtype=torch.bfloat16)
    b.q[:, :, 0] = (0.25 + 8 * torch.rand(n, heads, generator=g)).bfloat16()       # one product a score: exact in 32 bits
    b.k[0].zero_()
    b.k[0][1::2, :, 0] = -1.0
    b.v[0][0::2] = 1.0
    b.v[0][1::2] = -torch.exp2(torch.linspace(-0.5, 3.5, dim)).bfloat16()
    at = torch.arange(kv)
    ops.paged_cache_write(b.k[0].cuda(), b.v[0].cuda(), (b.table[0][at // 16].long() * 16 + at % 16).cuda(), **names(b.cache))
    out, _ = b.call(causal=False, scale=scale)
    torch.cuda.synchronize()
    k, v = b.held(0, "k")[:, 0], b.held(0, "v")[:, 0]
    x = torch.einsum("nhd,kd->nhk", b.q.double(), k) * scale
    p = torch.exp(x - x.amax(2, keepdim=True))
    want, share = (p @ v) / p.sum(2, keepdim=True), (p @ v.abs()) / p.sum(2, keepdim=True)
    # p: fp16 for an E4M3 cache; for a bf16 cache two bf16 in the split-KV kernel (half a step of what half a step leaves), one in the
    # tensor-core kernel.  Everything else is 32-bit: the score's three roundings (|x| <= 4 in units of log2), 2^x (2^-22), sums of 200
    bits = 2.0 ** -11 if fp8 else 2.0 ** -8 if kernel == "chunk" else 2.0 ** -16
    bound = 2.0 ** -8 * want.abs() + (bits + 2.0 ** -17) * share
    err = (out.double().cpu() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())
    if fp8 or kernel != "chunk":                                     # one bf16 would not pass
        rough = (p.bfloat16().double() @ v) / p.sum(2, keepdim=True)
        assert ((rough - want).abs() > 2 * (2.0 ** -8 * want.abs() + (bits + 2.0 ** -17) * share)).any()


# ------------------------------------------------------------------------------------------------------ nothing to attend to
def test_no_sequences_and_tables_without_columns():
    """An empty batch is not an error, for the attention as for the read-back: every row is one of no sequence.  With a table
    without columns the sequences' rows see nothing, and only the rows of no sequence stay as they are in what is given."""
    import cudaop_b200 as ops
    cache = names(empty_cache(3, 2, 16, 64, True))

    def ints(*x, shape=None):
        return torch.tensor(x, dtype=torch.int32, device="cuda").view(shape or (len(x),))
    q = torch.ones(5, 4, 64, dtype=torch.bfloat16, device="cuda")
    for table in (ints(shape=(0, 0)), ints(shape=(0, 3))):
        out, lse = ops.paged_attention(q, page_table=table, cu_q=ints(0), kv_lens=ints(), max_q=1, return_lse=True, **cache)
        assert out.shape == q.shape and (out == 0).all() and lse.shape == (5, 4) and (lse == -math.inf).all()
        given = torch.full_like(q, 3.0)
        out, lse = ops.paged_attention(q, page_table=table, cu_q=ints(0), kv_lens=ints(), max_q=1, return_lse=True, out=given, **cache)
        assert (given == 3.0).all() and (lse == -math.inf).all()
        assert ops.paged_attention(q[:0], page_table=table, cu_q=ints(0), kv_lens=ints(), max_q=1, **cache).shape == (0, 4, 64)
        k, v = ops.paged_cache_read(page_table=table, cu_kv=ints(0), total=4, **cache)
        assert k.shape == (4, 2, 64) and (k == 0).all() and (v == 0).all()
        kv = [torch.full((4, 2, 64), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        ops.paged_cache_read(page_table=table, cu_kv=ints(0), total=4, k_out=kv[0], v_out=kv[1], **cache)
        assert (kv[0] == 3.0).all() and (kv[1] == 3.0).all()
    table = ints(shape=(2, 0))
    given = torch.full_like(q, 3.0)
    out, lse = ops.paged_attention(q, page_table=table, cu_q=ints(0, 1, 3), kv_lens=ints(1, 7), max_q=2, return_lse=True, out=given, **cache)
    assert (given[:3] == 0).all() and (given[3:] == 3.0).all() and (lse == -math.inf).all()
    out, lse = ops.paged_attention(q, page_table=table, cu_q=ints(0, 1, 3), kv_lens=ints(1, 7), max_q=2, return_lse=True, **cache)
    assert (out == 0).all() and (lse == -math.inf).all()
    kv = [torch.full((4, 2, 64), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    ops.paged_cache_read(page_table=table, cu_kv=ints(0, 1, 3), total=4, k_out=kv[0], v_out=kv[1], **cache)
    for t in kv:
        assert (t[:3] == 0).all() and (t[3:] == 3.0).all()
    k, v = ops.paged_cache_read(page_table=table, cu_kv=ints(0, 1, 3), total=4, **cache)
    assert (k == 0).all() and (v == 0).all()
    torch.cuda.synchronize()
    assert ops.status() == 0


# ------------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    import cudaop_b200 as ops
    b = Batch([2, 1], [20, 10], 4, 2, 64, 16, True)
    c = names(b.cache)
    dev = dict(page_table=b.table.cuda(), cu_q=b.cu.cuda(), kv_lens=torch.tensor(b.kv, dtype=torch.int32).cuda(), max_q=2)
    q = b.q.cuda()

    def refused(**change):
        args = {**c, **dev, **{k: v for k, v in change.items() if k != "q"}}
        with pytest.raises(ValueError):
            ops.paged_attention(change.get("q", q), **args)
    refused(q=q.float())
    refused(q=q.cpu())
    refused(q=q[:, :3])                                              # 3 heads on 2
    refused(q=torch.cat([q, q], 2))                                  # head_dim
    refused(q=torch.cat([q, q], 2)[:, :, ::2])                       # not contiguous
    refused(q=torch.zeros(3, 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[:, 1:].unflatten(1, (4, 64)))      # alignment
    refused(k_scale=None)
    refused(v_scale=c["v_scale"][:1])
    refused(k_cache=c["k_cache"].float())
    refused(k_cache=c["k_cache"][:, :, :8].contiguous(), v_cache=c["v_cache"][:, :, :8].contiguous())            # page size 8
    refused(k_cache=c["k_cache"].transpose(1, 2))
    refused(page_table=dev["page_table"].long())
    refused(page_table=dev["page_table"].cpu())
    refused(page_table=dev["page_table"][:1].contiguous())
    refused(cu_q=dev["cu_q"][:2].contiguous())
    refused(kv_lens=dev["kv_lens"].float())
    refused(max_q=0)
    refused(window=-1)
    refused(window=4, causal=False)
    refused(scale=NAN)
    refused(out=torch.zeros(3, 4, 64, device="cuda"))
    refused(out=torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda"))
    kv = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(3).cuda()
    for bad in (dict(k=kv.float()), dict(v=kv[:2]), dict(slots=slots.int()), dict(slots=slots[:2]), dict(slots=slots.cpu()), dict(k=kv[:, :1], v=kv[:, :1])):
        with pytest.raises(ValueError):
            ops.paged_cache_write(**{**dict(k=kv, v=kv, slots=slots), **bad, **c})
    cu = torch.tensor([0, 20, 30], dtype=torch.int32, device="cuda")
    for bad in (dict(total=-1), dict(cu_kv=cu[:2].contiguous()), dict(cu_kv=cu.long()), dict(k_out=kv), dict(k_out=kv, v_out=kv)):
        with pytest.raises(ValueError):
            ops.paged_cache_read(**{**dict(page_table=dev["page_table"], cu_kv=cu, total=30), **bad, **c})
    # nothing to do is not an error
    ops.paged_cache_write(kv[:0], kv[:0], slots[:0], **c)
    assert ops.paged_cache_read(page_table=dev["page_table"], cu_kv=cu, total=0, **c)[0].shape == (0, 2, 64)
    assert ops.paged_attention(q[:0], **{**c, **dev}).shape == (0, 4, 64)
    torch.cuda.synchronize()
    assert ops.status() == 0
