"""The 4-bit cache without a GPU: the row format's own properties, the kernels' division-free rounding
restated, and what every entry point refuses."""

import numpy as np
import pytest
import torch

import nano_vllm_b200 as lib
from nano_vllm_b200 import _native as nv
from nano_vllm_b200.layers.qk_prep import qk_norm_rope_write
from nano_vllm_b200.layers.rotary_embedding import RoPE
from u4_reference import GROUP, pack, quantise, values64

MAGIC = np.float32(12582912.0)


def _rows(kind, dtype, n=400, D=128, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(n, D, generator=gen)
    if kind == "offset":
        x = x * 0.01 + 30 * torch.randn(n, 1, generator=gen)
    elif kind == "tiny":
        x = x * 2.0 ** -22
    elif kind == "wide":
        x = x * torch.exp(4 * torch.randn(n, 1, generator=gen))
    elif kind == "constant":
        x = torch.ones(n, D) * torch.randn(n, 1, generator=gen)
    elif kind == "ties":
        x = torch.randint(-30, 31, (n, D), generator=gen).float() / 2
    return x.to(dtype)


@pytest.mark.parametrize("kind", ["normal", "offset", "tiny", "wide", "constant", "ties"])
@pytest.mark.parametrize("dtype,scale", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                         (torch.float32, torch.bfloat16), (torch.float32, torch.float16)])
def test_no_value_is_off_by_more_than_half_a_step(kind, dtype, scale):
    x = _rows(kind, dtype)
    codes, s, z = quantise(x, scale)
    v = values64(*pack(codes, s, z, scale))
    step = torch.from_numpy(np.repeat(s, GROUP, -1)).double()
    # half a step, and the fp32 roundings of x - z, of the span and of the quotient (each 2^-24 of
    # what it rounds: x - z is up to 15 steps, so 15 * 3 * 2^-24 of a step) and of z's size
    slack = step * 45 * 2.0 ** -24 + x.double().abs() * 2.0 ** -24
    groups = x.view(-1, 2, GROUP)
    held = torch.isfinite(groups).all(-1, keepdim=True) & (groups.amin(-1, keepdim=True).float() >= -torch.finfo(scale).max)
    held = held.expand(-1, -1, GROUP).reshape(x.shape)
    assert ((v - x.double()).abs() <= step / 2 + slack)[held].all() and held.float().mean() > 0.9
    assert v[~held].isnan().all()  # beyond float16's numbers


@pytest.mark.parametrize("kind", ["normal", "offset", "wide", "ties"])
def test_guarded_product_rounds_like_the_quotient(kind):
    """u4_code_fast: t = fl(fl(x - z) * fl(1 / s)) rounded through the shifter equals rint of the
    quotient wherever t is 2^-14 from every half-integer; elsewhere the kernels divide."""
    for dtype in (torch.bfloat16, torch.float16):
        x = _rows(kind, dtype, 3000)
        codes, s, z = quantise(x, dtype)
        g = x.float().numpy().reshape(-1, 2, GROUP)
        some = s > 0
        d = (g - z[..., None])[some]
        r = (np.float32(1) / s[some])[:, None]
        t = d * r
        f = t + MAGIC
        sure = np.abs(t - (f - MAGIC)) < np.float32(0.5 - 2.0 ** -14)
        q = np.clip(f.view(np.int32) - 0x4B400000, 0, 15)
        want = codes.reshape(-1, 2, GROUP)[some]
        assert np.array_equal(q[sure], want[sure])
        assert sure.mean() > (0.5 if kind == "ties" else 0.9)


def test_groups_that_cannot_be_held_are_nan():
    x = torch.randn(6, 128)
    x[0, 3], x[1, 70], x[2, 0], x[2, 1] = float("nan"), float("inf"), 3e38, -3e38
    x[3, 5] = -float("inf")
    codes, s, z = quantise(x, torch.bfloat16)
    v = values64(*pack(codes, s, z, torch.bfloat16))
    bad = v.isnan().view(6, 2, GROUP)
    assert bad[0, 0].all() and bad[1, 1].all() and bad[2, 0].all() and bad[3, 0].all()
    assert bad.sum() == 4 * GROUP


def _pools(P=4, Hkv=2, ps=16, D=128, dtype=torch.bfloat16):
    kp = torch.zeros(P, Hkv, ps, D // 2, dtype=torch.uint8)
    ks = torch.zeros(P, Hkv, ps, D // 32, dtype=dtype)
    return kp, kp.clone(), ks, ks.clone()


def test_pool_asks_for_its_group_size():
    with pytest.raises(ValueError, match="kv_group_size=64"):
        lib.TinyKvPagedPool(kv_bits=4)
    with pytest.raises(ValueError, match="kv_group_size=64"):
        lib.TinyKvPagedPool(kv_bits=4, kv_group_size=32)
    with pytest.raises(ValueError, match="kv_bits=4"):
        lib.TinyKvPagedPool(kv_bits=8, kv_group_size=64)
    assert lib.TinyKvPagedPool(kv_bits=4, kv_group_size=64).kv_bits == 4


def test_pool_storage_on_the_host():
    """Storage is laid out by the first keys: half-width uint8 rows, a scale and an offset a group; growth
    keeps what was there."""
    for dtype, held in ((torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16)):
        pool = lib.TinyKvPagedPool(page_size=4, kv_bits=4, kv_group_size=64, device="cpu")
        pool.allocate_page()
        pool.grow()
        pool._ensure_page_storage(torch.zeros(1, 2, 1, 128, dtype=dtype))
        assert pool.key_pages.shape == (1, 2, 4, 64) and pool.key_pages.dtype == torch.uint8
        assert pool.value_scales.shape == (1, 2, 4, 4) and pool.value_scales.dtype == held
        pool.key_pages.fill_(7)
        pool.key_scales.fill_(2)
        pool.allocate_page()
        pool.grow()
        pool._ensure_page_storage(torch.zeros(1, 2, 1, 128, dtype=dtype))
        assert pool.key_pages.shape[0] == 2 and (pool.key_pages[0] == 7).all() and (pool.key_scales[0] == 2).all()
        assert (pool.key_pages[1] == 0).all() and (pool.key_scales[1] == 0).all()
    with pytest.raises(ValueError, match="64 or 128"):
        pool = lib.TinyKvPagedPool(page_size=4, kv_bits=4, kv_group_size=64, device="cpu")
        pool.allocate_page()
        pool.grow()
        pool._ensure_page_storage(torch.zeros(1, 2, 1, 80))
    pool = lib.TinyKvPagedPool(page_size=4, kv_bits=4, kv_group_size=64, device="cpu", reserve_pages=8)
    pool.allocate_page()
    pool.grow()
    pool._ensure_page_storage(torch.zeros(1, 2, 1, 64, dtype=torch.float16))
    assert pool.key_pages.shape == (1, 2, 4, 32) and pool.key_scales.shape == (1, 2, 4, 2)


@pytest.mark.parametrize("change,words", [
    (dict(D=80), "64 or 128"),
    (dict(values=torch.zeros(4, 2, 16, 64, dtype=torch.int8)), "uint8"),
    (dict(scales=None), "need key_scales"),
    (dict(scales=torch.zeros(4, 2, 16, 1, dtype=torch.bfloat16)), "a scale and an offset"),
    (dict(scales=torch.zeros(4, 2, 16, 4, dtype=torch.float32)), "float16 or both bfloat16"),
    (dict(scales=torch.zeros(4, 2, 16, 4, dtype=torch.float16)), "float16 or both bfloat16"),
    (dict(scales=torch.zeros(4, 2, 16, 8, dtype=torch.bfloat16)[..., ::2]), "contiguous"),
])
def test_refused_pools(change, words):
    kp, vp, ks, vs = _pools()
    with pytest.raises(RuntimeError, match=words):
        nv.require_u4("op", change.get("D", 128), kp, change.get("values", vp), change.get("scales", ks), vs)


def test_calls_without_a_gpu_are_refused():
    kp, vp, ks, vs = _pools()
    q = torch.zeros(1, 4, 1, 128, dtype=torch.bfloat16)
    bt, cl = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA device"):
        lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs)
    with pytest.raises(RuntimeError, match="CUDA device"):
        lib.read_slots(torch.zeros(1, dtype=torch.int64), kp, vp, ks, vs)
    rows = torch.zeros(1, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA device"):
        lib.write_slots(rows, rows, torch.zeros(1, dtype=torch.int64), kp, vp, ks, vs)
    x = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA device"):
        qk_norm_rope_write(x, x, x, None, None, RoPE(128, 8), torch.zeros(1, 1, dtype=torch.int32), kp, vp,
                           torch.zeros(1, dtype=torch.int64), key_scales=ks, value_scales=vs)
    for more in (dict(window=4), dict(sinks=1), dict(key_mass=torch.zeros(1, 2, 64))):
        with pytest.raises(NotImplementedError, match="4-bit"):
            lib.paged_attention(q, kp, vp, bt, cl, 16, ks, vs, **more)


def _paged(**kw):
    a = dict(q=None, kp=None, ks=None, sdt=nv.NVM_BF16, D=128, P=4, Hkv=2, ps=16, mp=0, B=1)
    a.update(kw)
    return nv.lib().nvm_paged_attention(a["q"], nv.NVM_BF16, a["kp"], a["kp"], nv.NVM_U4, a["ks"], a["ks"], a["sdt"], None, None,
                                        None, nv.NVM_BF16, a["B"], 4, a["Hkv"], 1, a["D"], a["P"], a["ps"], a["mp"], 0.1, 1, None,
                                        0, None)


def test_c_entry_points_refuse():
    """Host checks only: nothing is launched."""
    L = nv.lib()
    message = lambda: L.nvm_last_error().decode()  # noqa: E731
    assert _paged(D=96) == -2 and "64 or 128" in message()
    assert _paged(sdt=nv.NVM_F32) == -1 and "float16 or bfloat16" in message()
    assert _paged(P=2 ** 30, ps=16) == -2 and "2^32" in message()
    assert _paged(mp=4) == -1 and "pages and scales" in message()
    assert _paged(mp=4, kp=8, ks=16) == -1 and "16-byte" in message()
    assert _paged(mp=4, kp=16, ks=4) == -1 and "8-byte" in message()
    assert _paged(mp=4, kp=16, ks=16) == -1 and "null tensor pointer" in message()
    assert _paged(B=0) == 0
    assert L.nvm_paged_attention_window(None, 2, None, None, nv.NVM_U4, None, None, 2, None, None, None, 2, 1, 4, 2, 1, 128, 4, 16,
                                        4, 0.1, 1, 8, 0, None, 0, 0, 0, None, 0, None) == -2
    assert "4-bit" in message()
    assert L.nvm_paged_attention_window_workspace_size(1, 4, 2, 1, 128, 16, 4, nv.NVM_U4, 8, 0, 0) == 0
    write = lambda **k: L.nvm_reshape_and_cache(*[16] * 2, k.get("dt", 2), 0, 0, *[k.get("kp", 16)] * 2, nv.NVM_U4,  # noqa: E731
                                                *[k.get("ks", 16)] * 2, k.get("sdt", 2), 16, k.get("T", 1), k.get("H", 2),
                                                k.get("D", 128), 4, 16, None)
    assert write(dt=3) == -1
    assert write(D=32) == -2 and "64 or 128" in message()
    assert write(sdt=0) == -1 and write(ks=None) == -1 and write(kp=8) == -1
    assert write(T=2 ** 31) == -2 and "too many rows" in message()
    read = lambda **k: L.nvm_read_slots(*[k.get("kp", 16)] * 2, k.get("kv", nv.NVM_U4), *[k.get("ks", 16)] * 2,  # noqa: E731
                                        k.get("sdt", 2), 16, k.get("k", 16), 16, k.get("out", 2), k.get("T", 1), 2, k.get("D", 128), 4, 16,
                                        None)
    assert read(out=3) == -1 and read(kv=4) == -1 and read(D=32) == -2 and read(ks=None) == -1 and read(kp=8) == -1
    assert read(kv=nv.NVM_I8, ks=None) == -1 and read(T=2 ** 31) == -2 and read(T=0) == 0 and read(D=0) == -1
    assert read(k=8) == -1 and "16-byte" in message()
    prep = lambda **k: L.nvm_qk_norm_rope_write(16, 16, 16, 2, 512, 256, k.get("wq", None), k.get("wk", None), 1e-6, 16,  # noqa: E731
                                                16, 8, 0, 16, 16, 1, 16, 16, nv.NVM_U4, k.get("ks", 16), 16, k.get("sdt", 2), 16,
                                                k.get("T", 0), 4, 2, 128, 4, 16, None)
    assert prep() == 0  # no tokens
    assert prep(wq=16) == -1 and "both or not at all" in message()
    assert prep(sdt=1) == -1 and prep(ks=None) == -1 and prep(ks=4) == -1




def test_quotient_by_fifteen_is_rounded_as_the_division():
    """The kernels' over15 restated, for every fp32 mantissa (the exponent only shifts both): with y = fl(1/15)
    and q = fl(x y), fl(fl(x - 15 q) y + q) is fl(x / 15).  x - 15 q is exact in 64 bits; the last step is an
    addition of numbers 2^20 apart, whose 64-bit sum is rounded to fp32 unless it is a tie of that rounding,
    and those are none (an exact tie of x / 15 would need 15 to divide a power of two)."""
    y = np.float32(1) / np.float32(15)
    m = np.arange(1 << 23, 1 << 24, dtype=np.int64)
    x = m.astype(np.float32)
    q = x * y
    r = (x.astype(np.float64) - 15.0 * q.astype(np.float64)).astype(np.float32)
    got = (r.astype(np.float64) * np.float64(y) + q.astype(np.float64)).astype(np.float32)
    assert np.array_equal(got, x / np.float32(15))
