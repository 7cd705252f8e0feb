"""What the C ABI of the MXFP4 and paged-cache operators refuses, without a GPU: arguments are checked before any device
call, so the pointers here are never followed."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as g
    g.build()
    import cudaop_b200 as ops
    return ops.lib()


P = 1 << 20                     # an aligned address that is never read


def attention(lib, **change):
    a = dict(q=P, kc=P, vc=P, ks=P, vs=P, table=P, cu=P, kv=P, out=P, lse=None, seqs=2, tokens=3, heads=8, kv_heads=2, dim=128, qs=1024,
             qh=128, max_q=2, max_pages=4, pages=10, page=16, fp8=1, scale=1.0, causal=1, window=0, rest=1, ws=P, stream=None)
    a.update(change)
    return lib.b200q_paged_attention(*a.values())


BAD = [dict(q=None), dict(kc=None), dict(vs=None), dict(cu=None), dict(ws=None), dict(q=P + 2), dict(kc=P + 8), dict(out=P + 4), dict(ks=P + 4),
       dict(ws=P + 8), dict(seqs=0), dict(tokens=0), dict(heads=7), dict(heads=0), dict(kv_heads=0), dict(dim=96), dict(dim=256), dict(page=8),
       dict(page=48), dict(page=256), dict(qs=1020), dict(qh=100), dict(max_q=0), dict(max_pages=0), dict(pages=0), dict(window=-1),
       dict(window=8, causal=0), dict(scale=float("nan")), dict(max_pages=2 ** 27, page=16), dict(pages=2 ** 27, page=16),
       dict(tokens=2 ** 28, heads=8), dict(seqs=8193)]


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_attention(lib, bad):
    assert attention(lib, **bad) == 1


WRITE = dict(k=P, v=P, slots=P, kc=P, vc=P, ks=P, vs=P, tokens=4, heads=2, dim=64, a=128, b=128, c=64, d=64, pages=4, page=16, fp8=1, stream=None)
READ = dict(kc=P, vc=P, ks=P, vs=P, table=P, cu=P, k=P, v=P, seqs=2, total=9, heads=2, dim=64, max_pages=3, pages=4, page=16, fp8=1, rest=1, stream=None)


@pytest.mark.parametrize("bad", [dict(k=None), dict(slots=None), dict(ks=None), dict(k=P + 8), dict(vc=P + 8), dict(slots=P + 4), dict(tokens=0),
                                 dict(heads=0), dict(dim=32), dict(page=20), dict(pages=0), dict(a=4), dict(d=12)], ids=str)
def test_write(lib, bad):
    assert lib.b200q_paged_cache_write(*{**WRITE, **bad}.values()) == 1


@pytest.mark.parametrize("bad", [dict(k=None), dict(table=None), dict(vs=None), dict(v=P + 8), dict(kc=P + 4), dict(seqs=0), dict(total=0), dict(heads=0),
                                 dict(dim=100), dict(page=0), dict(pages=0), dict(max_pages=0)], ids=str)
def test_read(lib, bad):
    assert lib.b200q_paged_cache_read(*{**READ, **bad}.values()) == 1


@pytest.mark.parametrize("bad", [dict(a=None), dict(sfb=None), dict(c=None), dict(m=0), dict(n=0), dict(k=0), dict(k=48), dict(a=P + 8), dict(sfa=P + 4)], ids=str)
def test_mxfp4_product(lib, bad):
    a = dict(a=P, sfa=P, b=P, sfb=P, c=P, m=4, n=8, k=64, stream=None)
    assert lib.b200q_gemm_mxfp4_blocked(*{**a, **bad}.values()) == 1


@pytest.mark.parametrize("bad", [dict(x=None), dict(q=None), dict(sf=None), dict(rows=0), dict(cols=16), dict(x=P + 8), dict(q=P + 2), dict(sf=P + 8)], ids=str)
def test_mxfp4_quantiser(lib, bad):
    a = dict(x=P, q=P, sf=P, rows=4, cols=64, stream=None)
    assert lib.b200q_quant_rows_mxfp4(*{**a, **bad}.values()) == 1


def test_sizes(lib):
    assert lib.b200q_paged_attention_workspace_bytes(96) == 0
    assert lib.b200q_gemm_mxfp4_workspace_bytes(3, 130, 160) == (1 + 2) * 2 * 512
    assert lib.b200q_gemm_mxfp4_workspace_bytes(3, 130, 48) == 0
