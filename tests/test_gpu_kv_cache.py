"""kv_cache_write / kv_cache_read: bytes and scales against ROWWISE quantize_fp8
and its definition, slots, strides, types, untouched slots, offsets past 32 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

E4, E5, BF, FH = torch.float8_e4m3fn, torch.float8_e5m2, torch.bfloat16, torch.float16


def _ops():
    import primus_turbo.pytorch as turbo

    return turbo.ops


def _cache(P, H, page, D, dtype):
    kv = [torch.full((P, H, page, D), 3.0, device="cuda").to(dtype) for _ in range(2)]
    sc = [torch.full((P, H, page), 7.0, device="cuda") for _ in range(2)] if dtype in (E4, E5) else [None, None]
    return kv + sc


def _rows(pool, slots, page):
    s = slots.cpu().long()
    x = pool.cpu()
    x = x.view(torch.uint8) if x.element_size() == 1 else x
    return x[s // page, :, s % page]


@pytest.mark.parametrize("dtype", [BF, FH, torch.float32])
@pytest.mark.parametrize("cache", [E4, E5])
@pytest.mark.parametrize("T,H,D,page", [(1, 1, 16, 1), (5, 3, 48, 7), (33, 8, 128, 16), (129, 2, 64, 64), (70, 5, 256, 48)])
def test_write_is_rowwise_quantization(dtype, cache, T, H, D, page):
    from primus_turbo.pytorch.core.low_precision import ScalingGranularity

    ops = _ops()
    g = torch.Generator().manual_seed(T * D)
    P = -(-T // page) + 2
    slots = torch.randperm(P * page, generator=g)[:T].cuda()
    k, v = ((torch.randn(T, H, D, generator=g) * 3).to(dtype).cuda() for _ in range(2))
    k[0, 0] = 0  # a row of zeros
    kc, vc, ks, vs = _cache(P, H, page, D, cache)
    ops.kv_cache_write(k, v, kc, vc, slots, ks, vs)
    for x, pool, sc in ((k, kc, ks), (v, vc, vs)):
        q, s = ops.quantize_fp8(x.reshape(T * H, D), cache, ScalingGranularity.ROWWISE, axis=-1)
        assert torch.equal(_rows(pool, slots, page), q.view(torch.uint8).view(T, H, D).cpu())
        assert torch.equal(_rows(sc, slots, page), s.view(T, H).cpu())
        rest = torch.ones(P * page, dtype=torch.bool)
        rest[slots.cpu()] = False
        assert bool((pool.cpu().float().permute(0, 2, 1, 3).reshape(P * page, H, D)[rest] == 3.0).all())
        assert bool((sc.cpu().permute(0, 2, 1).reshape(P * page, H)[rest] == 7.0).all())
    for out in (BF, FH, torch.float32):
        rk, rv = ops.kv_cache_read(kc, vc, slots, ks, vs, out_dtype=out)
        for y, pool, sc in ((rk, kc, ks), (rv, vc, vs)):
            want = (_rows(pool, slots, page).view(cache).float() * _rows(sc, slots, page)[..., None]).to(out)
            assert y.dtype == out and torch.equal(y.cpu(), want)


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("T,H,D,page", [(3, 1, 16, 2), (65, 4, 80, 16), (40, 2, 256, 5)])
def test_sixteen_bit_cache_moves_bits(dtype, T, H, D, page):
    ops = _ops()
    g = torch.Generator().manual_seed(T)
    P = -(-T // page) + 1
    slots = torch.randperm(P * page, generator=g)[:T].to(torch.int32).cuda()
    bits = torch.randint(-32768, 32768, (2, T, H, D), generator=g, dtype=torch.int16).cuda()  # NaN and infinities too
    kc, vc, _, _ = _cache(P, H, page, D, dtype)
    ops.kv_cache_write(bits[0].view(dtype), bits[1].view(dtype), kc, vc, slots)
    rk, rv = ops.kv_cache_read(kc, vc, slots, out_dtype=dtype)
    assert torch.equal(rk.view(torch.int16), bits[0]) and torch.equal(rv.view(torch.int16), bits[1])


def test_special_values_as_rowwise():
    from primus_turbo.pytorch.core.low_precision import ScalingGranularity

    ops = _ops()
    x = torch.randn(6, 2, 64, generator=torch.Generator().manual_seed(3)).to(BF)
    x[0, 0, 3], x[1, 1, 5], x[2, 0, 0], x[3] = float("nan"), float("inf"), -float("inf"), float("nan")
    x[4, 0] = 1e-30
    x = x.cuda()
    for cache in (E4, E5):
        kc, vc, ks, vs = _cache(2, 2, 4, 64, cache)
        ops.kv_cache_write(x, x, kc, vc, torch.arange(6, device="cuda"), ks, vs)
        q, s = ops.quantize_fp8(x.reshape(12, 64), cache, ScalingGranularity.ROWWISE, axis=-1)
        at = torch.arange(6)
        assert torch.equal(_rows(kc, at, 4), q.view(torch.uint8).view(6, 2, 64).cpu())
        assert torch.equal(_rows(vs, at, 4), s.view(6, 2).cpu())


@pytest.mark.parametrize("cache", [E4, BF])
def test_strides_and_skipped_slots(cache):
    """Slices of a projection's output, offsets that allow no 16-byte loads, a
    transposed tensor; slots outside the pool are skipped and read as zeros."""
    ops = _ops()
    T, H, D, page, P = 37, 4, 64, 16, 4
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn(T, 3 * H * D + 3, generator=g).to(BF).cuda()
    last = torch.randn(D, H, T, generator=g).to(BF).cuda().permute(2, 1, 0)
    slots = torch.randperm(P * page, generator=g)[:T]
    slots[3], slots[7], slots[20] = -1, P * page, 2 ** 40
    slots = slots.cuda()
    for off, x in ((0, None), (1, None), (0, last)):
        k = qkv[:, off + H * D:off + 2 * H * D].view(T, H, D) if x is None else x
        v = qkv[:, off + 2 * H * D:off + 3 * H * D].view(T, H, D)
        a, b = _cache(P, H, page, D, cache), _cache(P, H, page, D, cache)
        ops.kv_cache_write(k, v, a[0], a[1], slots, a[2], a[3])
        ops.kv_cache_write(k.contiguous(), v.contiguous(), b[0], b[1], slots, b[2], b[3])
        for p, q in zip(a, b):
            assert p is None or torch.equal(p.view(torch.uint8), q.view(torch.uint8))
        rk, rv = ops.kv_cache_read(a[0], a[1], slots, a[2], a[3], out_dtype=BF)
        for y, x0 in ((rk, k), (rv, v)):
            out = torch.tensor([3, 7, 20])
            assert bool((y.cpu()[out] == 0).all())
            keep = torch.ones(T, dtype=torch.bool)
            keep[out] = False
            # half an fp8 step of the row's largest value
            d = (y.float() - x0.float()).abs().cpu()[keep]
            assert bool((d <= x0.float().abs().amax(-1, keepdim=True).cpu()[keep] * (2.0 ** -4 if cache == E4 else 0.0)).all())


def test_no_tokens_and_no_pages():
    ops = _ops()
    kc, vc, ks, vs = _cache(2, 2, 4, 32, E4)
    x = torch.empty(0, 2, 32, dtype=BF, device="cuda")
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    ops.kv_cache_write(x, x, kc, vc, none, ks, vs)
    k, v = ops.kv_cache_read(kc, vc, none, ks, vs)
    assert k.shape == v.shape == (0, 2, 32)
    e = _cache(0, 2, 4, 32, E4)
    x = torch.ones(3, 2, 32, dtype=BF, device="cuda")
    slots = torch.arange(3, device="cuda")
    ops.kv_cache_write(x, x, e[0], e[1], slots, e[2], e[3])
    k, v = ops.kv_cache_read(e[0], e[1], slots, e[2], e[3])
    assert not bool(k.any()) and not bool(v.any())


def test_offsets_past_32_bits():
    """Pools of more than 2^32 bytes: the last pages are where they belong."""
    ops = _ops()
    P, H, page, D = 4200, 8, 512, 256  # 4.4e9 bytes a pool
    kc, vc = (torch.zeros((P, H, page, D), dtype=torch.uint8, device="cuda").view(E4) for _ in range(2))
    ks, vs = (torch.ones((P, H, page), device="cuda") for _ in range(2))
    slots = torch.tensor([P * page - 1, (P - 1) * page, 5, (P // 2) * page + 3], device="cuda")
    x = torch.randn(4, H, D, generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    ops.kv_cache_write(x, -x, kc, vc, slots, ks, vs)
    k, v = ops.kv_cache_read(kc, vc, slots, ks, vs, out_dtype=torch.float32)
    want = kc.view(torch.uint8)[slots // page, :, slots % page].view(E4).float() * ks[slots // page, :, slots % page][..., None]
    assert torch.equal(k, want) and torch.equal(v, -want)
    assert bool(((k - x.float()).abs() <= 2.0 ** -4 * x.float().abs().amax(-1, keepdim=True)).all())


def test_other_stream():
    ops = _ops()
    kc, vc, ks, vs = _cache(4, 2, 16, 128, E4)
    s = torch.cuda.Stream()
    x = torch.randn(64, 2, 128, device="cuda", dtype=BF)
    slots = torch.arange(64, device="cuda")
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = x * 2
        ops.kv_cache_write(y, y, kc, vc, slots, ks, vs)
        k, _ = ops.kv_cache_read(kc, vc, slots, ks, vs, out_dtype=torch.float32)
    torch.cuda.current_stream().wait_stream(s)
    assert bool(((k - 2 * x.float()).abs() <= 2.0 ** -4 * 2 * x.float().abs().amax(-1, keepdim=True)).all())
