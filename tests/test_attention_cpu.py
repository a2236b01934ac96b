"""CPU: what the attention operators refuse, before any launch, and the oracle's
own arithmetic (the 8-bit codes against torch's, the softmax against differences)."""
import importlib

import numpy as np
import pytest
import torch

from oracle import attention as A

L = importlib.import_module("10_20_b200.latent_attention")
K = importlib.import_module("10_20_b200.kv8")
BF = torch.bfloat16


def i32(*s):
    return torch.zeros(s, dtype=torch.int32)


def slots(**kw):
    a = dict(q=torch.zeros((2, 4, 576), dtype=BF), pool=torch.zeros((64, 1, 576), dtype=BF), req=None,
             ids=i32(2, 8), scale=0.1, latent=512)
    a.update(kw)
    return L.attend_slots(a["q"], a["pool"], a["req"], a["ids"], a["scale"], latent=a["latent"])


@pytest.mark.parametrize("bad,word", [
    (dict(), "CUDA"),
    (dict(q=torch.zeros((2, 4, 576))), "bfloat16"),
    (dict(q=torch.zeros((2, 576), dtype=BF)), "rows, heads"),
    (dict(pool=torch.zeros((64, 1, 576), dtype=torch.float16)), "q's type"),
    (dict(pool=torch.zeros((64, 2, 576), dtype=BF)), "slots, 1"),
    (dict(pool=torch.zeros((64, 1, 512), dtype=BF)), "slots, 1"),
    (dict(latent=500), "latent"),
    (dict(latent=256), "latent"),
    (dict(ids=torch.zeros((2, 8), dtype=torch.int64)), "int32"),
    (dict(ids=i32(3, 8)), "ids"),
    (dict(ids=i32(2, 16)[:, ::2]), "inner stride"),
    (dict(req=torch.zeros(8, dtype=torch.int64)), "request_slots"),
    (dict(q=torch.zeros((2, 4, 577), dtype=BF)[:, :, 1:]), "16-byte"),
    (dict(q=torch.zeros((2, 4, 580), dtype=BF)[:, :, :576]), "16-byte"),
    (dict(scale=float("nan")), "finite"),
    (dict(q=torch.zeros((2, 1025, 576), dtype=BF)), "heads"),
])
def test_attend_slots_refuses(bad, word):
    with pytest.raises(ValueError, match=word):
        slots(**bad)


@pytest.mark.parametrize("table,lens,word", [
    (i32(2, 3), i32(2), "CUDA"), (i32(1, 3), i32(2), "table"), (i32(2, 3), i32(3), "lens"),
    (i32(2, 6)[:, ::2], i32(2), "inner stride"), (i32(2, 3), torch.zeros(2, dtype=torch.int64), "lens"),
    (torch.zeros((2, 3)), i32(2), "table"),
])
def test_attend_pages_refuses(table, lens, word):
    with pytest.raises(ValueError, match=word):
        L.attend_pages(torch.zeros((2, 4, 576), dtype=BF), torch.zeros((64, 1, 576), dtype=BF), table, lens, 0.1)


@pytest.mark.parametrize("bad,word", [
    (dict(), "CUDA"),
    (dict(q=torch.zeros((8, 4, 128), dtype=BF)), "q:"),
    (dict(k=torch.zeros((8, 3, 128), dtype=BF)), "k, v"),
    (dict(v=torch.zeros((8, 4, 64), dtype=BF)), "k, v"),
    (dict(v=torch.zeros((8, 4, 128), dtype=torch.float16)), "one type"),
    (dict(k_rope=torch.zeros((7, 64), dtype=BF)), "k_rope"),
    (dict(k_rope=torch.zeros((8, 68), dtype=BF)[:, :64]), "16-byte"),
    (dict(offsets=torch.zeros(3, dtype=torch.int64)), "offsets"),
    (dict(kv_offsets=i32(2)), "offsets"),
    (dict(scale=float("inf")), "finite"),
])
def test_attend_prompt_refuses(bad, word):
    a = dict(q=torch.zeros((8, 4, 192), dtype=BF), k=torch.zeros((8, 4, 128), dtype=BF),
             k_rope=torch.zeros((8, 64), dtype=BF), v=torch.zeros((8, 4, 128), dtype=BF), offsets=i32(3), scale=0.1,
             kv_offsets=None)
    a.update(bad)
    with pytest.raises(ValueError, match=word):
        L.attend_prompt(a["q"], a["k"], a["k_rope"], a["v"], a["offsets"], a["scale"], kv_offsets=a["kv_offsets"])


def cache(pages=4, heads=2):
    c = lambda: torch.zeros((pages, heads, 64, 128), dtype=torch.float8_e4m3fn)
    s = lambda: torch.ones((pages, heads))
    return [c(), s(), c(), s()]


@pytest.mark.parametrize("at,value,word", [
    (None, None, "CUDA"),
    (0, torch.zeros((4, 2, 64, 128), dtype=torch.uint8), "float8"),
    (2, torch.zeros((4, 3, 64, 128), dtype=torch.float8_e4m3fn), "k_cache"),
    (1, torch.ones((4, 3)), "k_scale"),
    (3, torch.ones((4, 2), dtype=torch.float16), "k_scale"),
])
def test_cache_refusals(at, value, word):
    c = cache()
    if at is not None:
        c[at] = value
    x = torch.zeros((5, 2, 128), dtype=BF)
    with pytest.raises(ValueError, match=word):
        K.store(*c, x, x, i32(1, 2), i32(1), i32(2))
    with pytest.raises(ValueError, match=word):
        K.attend(torch.zeros((1, 4, 128), dtype=BF), *c, i32(1, 2), i32(1), 0.1)


@pytest.mark.parametrize("kw,word", [
    (dict(k=torch.zeros((5, 2, 64), dtype=BF)), "k, v"), (dict(k=torch.zeros((5, 2, 128))), "k, v"),
    (dict(k=torch.zeros((5, 2, 132), dtype=BF)[..., :128]), "16-byte"), (dict(offsets=i32(3)), "offsets"),
    (dict(prefix=torch.zeros(1, dtype=torch.int64)), "prefix"), (dict(table=i32(2, 2)), "table"),
])
def test_store_refuses(kw, word):
    x = torch.zeros((5, 2, 128), dtype=BF)
    a = dict(k=x, v=x, table=i32(1, 2), prefix=i32(1), offsets=i32(2))
    a.update(kw)
    with pytest.raises(ValueError, match=word):
        K.store(*cache(), a["k"], a["v"], a["table"], a["prefix"], a["offsets"])


@pytest.mark.parametrize("kw,word", [
    (dict(q=torch.zeros((1, 3, 128), dtype=BF)), "multiple"), (dict(q=torch.zeros((1, 4, 64), dtype=BF)), "q:"),
    (dict(lens=i32(2)), "lens"), (dict(table=i32(2, 2)), "table"), (dict(scale=float("nan")), "finite"),
])
def test_attend_refuses(kw, word):
    a = dict(q=torch.zeros((1, 4, 128), dtype=BF), table=i32(1, 2), lens=i32(1), scale=0.1)
    a.update(kw)
    with pytest.raises(ValueError, match=word):
        K.attend(a["q"], *cache(), a["table"], a["lens"], a["scale"])


def test_entry_points_refuse_before_a_launch():
    """The C entry points' own checks: no device pointer is followed."""
    lib = importlib.import_module("10_20_b200._lib").lib()
    x = 1 << 20   # an aligned address that is never read

    def latent(dtype=1, q=x, qs=576, heads=4, dim=576, latent=512, count=64, lens=None, index=x, req=None, rows=2,
               work=x, size=1 << 30):
        return lib.v1x_latent_attention(q, qs * heads, qs, x, 64, 576, req, 8, index, count, count, lens, rows, heads, dim,
                                        latent, 0.1, dtype, x, x, work, size, None, None)

    for bad in (dict(dtype=0), dict(q=x + 2), dict(qs=577), dict(heads=0), dict(heads=1025), dict(dim=560),
                dict(latent=64, dim=64), dict(count=65, lens=x), dict(lens=x, req=x), dict(index=None), dict(q=None),
                dict(rows=1, count=65536, size=0), dict(rows=1, count=65536, work=x + 8),
                dict(rows=1 << 30, count=1 << 35)):
        assert latent(**bad) == -1, bad
        assert b"latent_attention" in lib.v1x_last_error()
    pr = [x, 768, 192, x, 512, 128, x, 64, x, 512, 128, x, x, 1, 8, 8, 4, 64, 0.1, 1, x, x, None, None]
    for at, v in ((19, 3), (17, 32), (6, None), (0, x + 8), (1, 769), (11, None), (20, None), (16, 0)):
        bad = list(pr)
        bad[at] = v
        assert lib.v1x_prompt_attention(*bad) == -1, (at, v)
        assert b"prompt_attention" in lib.v1x_last_error()
    st = [x, x, x, x, 4, 2, x, 256, 128, x, 256, 128, 1, 8, x, 2, 2, x, x, 1, None]
    for at, v in ((12, 0), (0, x + 4), (7, 255), (4, -1), (5, 0), (17, None), (1, None)):
        bad = list(st)
        bad[at] = v
        assert lib.v1x_kv8_store(*bad) == -1, (at, v)
        assert b"kv8_store" in lib.v1x_last_error()
    at_ = [x, 512, 128, x, x, x, x, 4, 2, x, 2, 2, x, 1, 4, 0.1, 1, x, x, x, 1 << 30, None, None]
    for at, v in ((16, 0), (14, 3), (0, x + 2), (1, 511), (12, None), (9, None), (17, None), (20, 0), (19, x + 8), (7, 1 << 25)):
        bad = list(at_)
        bad[at] = v
        assert lib.v1x_kv8_attend(*bad) == -1, (at, v)
        assert b"kv8_attend" in lib.v1x_last_error()


def test_oracle_codes_are_torchs():
    g = torch.Generator().manual_seed(1)
    x = torch.cat([torch.randn(20000, generator=g) * s for s in (0.003, 0.1, 3, 100, 300)])
    x = torch.cat([x, torch.tensor(A.E4M3[:127]).float(), torch.tensor((A.E4M3[:126] + A.E4M3[1:127]) / 2).float()])
    x = torch.cat([x, -x])
    want = x.clamp(-448, 448).to(torch.float8_e4m3fn)
    assert np.array_equal(A.e4m3_encode(x.double().numpy()), want.view(torch.uint8).numpy())
    assert np.array_equal(A.e4m3_decode(want.view(torch.uint8).numpy()), want.double().numpy())


@pytest.mark.parametrize("most,e", [(0.0, -40), (448.0, 0), (448.5, 1), (447.0, 0), (224.0, -1), (2.0 ** -60, -40),
                                    (1e30, 40), (1.75, -8), (1.7500001, -7)])
def test_oracle_scale(most, e):
    assert A.page_scale(most) == 2.0 ** e


def test_oracle_lse_is_the_outputs_potential():
    """d lse / d s_j = p_j: lse against central differences, the output from them."""
    rng = np.random.default_rng(3)
    q, k, v = rng.standard_normal((1, 6)), rng.standard_normal((9, 6)), rng.standard_normal((9, 4))
    out, lse, _, _ = A.softmax_rows(q, k, v, 0.7)
    p = np.zeros(9)
    for j in range(9):
        def at(step):
            kk = np.vstack([k, np.zeros((1, 6))])
            s = q @ k.T * 0.7
            s[0, j] += step
            return np.log(np.exp(s).sum()), kk
        p[j] = (at(1e-5)[0] - at(-1e-5)[0]) / 2e-5
    assert np.allclose(p @ v, out[0], atol=1e-8)
    assert abs(lse[0] - np.log(np.exp(q @ k.T * 0.7).sum())) < 1e-12
