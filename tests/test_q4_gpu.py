"""Projections in 4 bits (strim_pack_weights, strim_unpack_weights, strim_head_logits_packed)
against their formulas in float64.

The bounds: a stored scale or bias half a bf16 spacing (and a float32 rounding) from the
formula's; a code the nearest one for the stored scale and bias (half a step and a float32
rounding), unless it is clamped; a value read back exactly s q + b, rounded once. A logit: half
a spacing of its type, and 1e-6 of the sum of the absolute terms that the kernel adds, s (16 +
q) |x|, 16 s |x| and |b x|, for the float32 accumulation (tests/test_head_gpu.py has the same)."""
import ctypes

import pytest
import torch

import head_oracle as H
from strim_amd import _native as N
from strim_amd import ops

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def codes(q):
    sh = 4 * torch.arange(8, device="cuda", dtype=torch.int32)
    return ((q.words[..., None] >> sh) & 15).reshape(q.V, -1, q.group).double()


def values(q):
    s = q.scales.double()[..., None]
    if q.biases is None:
        return ((codes(q) - 8) * s).reshape(q.V, q.K)
    return (codes(q) * s + q.biases.double()[..., None]).reshape(q.V, q.K)


def spacing(x, bits):
    return torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -126))) - bits)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("V,K,group", [(1, 32, 32), (3, 64, 64), (5, 128, 128), (37, 96, 32),
                                       (130, 320, 64), (1001, 1280, 128), (77, 5120, 64)])
def test_pack_and_unpack(V, K, group, symmetric, dtype):
    print(f"[q4] pack V={V} K={K} group={group} {symmetric} {dtype}", flush=True)
    g = gen(V + K)
    w = torch.randn(V, K, device="cuda", generator=g)
    w *= torch.exp(torch.randn(V, 1, device="cuda", generator=g))
    w[V // 2, : group] = 0.25  # a constant group
    w[0, -group:] = 0.0
    w = w.to(dtype)
    q = ops.q4_pack(w, group, symmetric)
    wd = w.double().reshape(V, -1, group)
    lo, hi = wd.amin(-1), wd.amax(-1)
    s = q.scales.double()
    ideal = wd.abs().amax(-1) / 7 if symmetric else (hi - lo) / 15
    assert bool(((s - ideal).abs() <= (2.0 ** -8 + 2.0 ** -22) * ideal).all())
    if symmetric:
        assert q.biases is None
        base, off = torch.zeros_like(s), 8.0
    else:
        base, off = q.biases.double(), 0.0
        assert bool(((base - lo).abs() <= 2.0 ** -8 * lo.abs()).all())
    live = s > 0
    c = codes(q)
    exact = torch.where(live[..., None], (wd - base[..., None]) / s.clamp_min(1e-300)[..., None], 0.0) + off
    want = exact.clamp(0, 15)
    # (float32: the difference's rounding, up to 2^-24 of |bias| / scale steps)
    slack = 1e-5 + 2.0 ** -22 * (base.abs() / s.clamp_min(1e-300))[..., None]
    assert bool((((c - want).abs() <= 0.5 + slack) | ~live[..., None]).all())
    assert bool((c[~live] == off).all())
    for out in (torch.bfloat16, torch.float32):
        got, ref = ops.q4_unpack(q, out), values(q)
        if out == torch.float32:
            assert bool(((got.double() - ref).abs() <= 2.0 ** -24 * ref.abs()).all())
        else:
            assert torch.equal(got, ref.float().to(out))


def test_pack_strided_rows_and_non_finite_groups():
    buf = torch.randn(20, 200, device="cuda", generator=gen(4))
    w = buf[:, :128]
    a, b = ops.q4_pack(w, 64), ops.q4_pack(w.contiguous(), 64)
    assert torch.equal(a.words, b.words) and torch.equal(a.scales, b.scales)
    w = w.contiguous()
    w[3, 70], w[4, 1] = float("nan"), float("inf")
    for sym in (False, True):
        v = ops.q4_unpack(ops.q4_pack(w, 64, sym), torch.float32)
        bad = torch.zeros(20, 128, dtype=torch.bool, device="cuda")
        bad[3, 64:], bad[4, :64] = True, True
        assert bool(v[bad].isnan().all()) and bool(v[~bad].isfinite().all())


def weight(V, K, group, symmetric, seed):
    g = gen(seed)
    words = torch.randint(-2 ** 31, 2 ** 31, (V, K // 8), device="cuda", generator=g).to(torch.int32)
    s = (0.2 + torch.rand(V, K // group, device="cuda", generator=g)) / 16
    s *= torch.where(torch.rand(V, K // group, device="cuda", generator=g) < 0.1, -3.0, 1.0)
    b = None if symmetric else (-s * (7.5 + torch.randn(V, K // group, device="cuda", generator=g)))
    return ops.Q4Weight(words, s.to(torch.bfloat16), None if b is None else b.to(torch.bfloat16), group)


def check_logits(x, q, got, label):
    xd, w = x.double(), values(q)
    ref = xd @ w.T
    s = q.scales.double().abs()[..., None]
    amp = s * (32 + codes(q))
    amp = amp + (8 * s if q.biases is None else q.biases.double().abs()[..., None])
    tol = 1e-6 * (xd.abs() @ amp.reshape(q.V, q.K).T) + 1e-30
    tol += 0.5 * spacing(ref, 7) * 1.01 if got.dtype == torch.bfloat16 else 2.0 ** -24 * ref.abs()
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), f"{label}: {float((err / tol).max()):.3g} of the bound"


LOGITS = [(1, 32, 1, 32), (1, 64, 15, 64), (1, 128, 17, 128), (2, 96, 33, 32), (3, 192, 100, 64),
          (4, 1024, 129, 32), (5, 1088, 250, 64), (8, 2048, 300, 64), (9, 384, 77, 128),
          (15, 4096, 513, 128), (16, 640, 257, 64), (17, 5120, 1000, 64), (31, 1152, 90, 128),
          (32, 8192, 300, 64), (33, 1056, 130, 32), (48, 5120, 700, 64), (49, 320, 64, 64),
          (63, 2560, 200, 128), (64, 5120, 999, 32), (65, 256, 40, 64), (130, 512, 70, 32),
          (1, 5120, 5000, 64), (1, 20480, 140, 64), (6, 12800, 64, 128), (1, 9216, 2100, 32),
          (20, 20480, 50, 32), (3, 1152, 500, 64), (7, 1152, 333, 32), (2, 1280, 77, 128),
          (6, 2560, 4000, 64), (12, 1280, 9000, 64), (24, 1088, 33_000, 64), (64, 1024, 33_000, 128),
          (50, 512, 70_003, 32), (10, 576, 90_000, 64), (64, 640, 160_001, 64)]


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("B,K,V,group", LOGITS)
def test_logits(B, K, V, group, symmetric):
    print(f"[q4] logits B={B} K={K} V={V} group={group} {symmetric}", flush=True)
    q = weight(V, K, group, symmetric, seed=B + K + V)
    x = (2.0 * torch.randn(B, K, device="cuda", generator=gen(B))).to(torch.bfloat16)
    for dt in (torch.bfloat16, torch.float32):
        got = ops.head_logits_q4(x, q, out_dtype=dt)
        check_logits(x, q, got, f"B={B} K={K} V={V} group={group} {dt}")


def test_logits_many_row_tiles():
    """More row tiles than the workgroups in flight, a row's tile partly past the vocabulary."""
    for B in (1, 7, 30, 64):
        print(f"[q4] many tiles B={B}", flush=True)
        q = weight(70_001, 256, 64, False, seed=B)
        x = torch.randn(B, 256, device="cuda", generator=gen(B)).to(torch.bfloat16)
        check_logits(x, q, ops.head_logits_q4(x, q), f"B={B}")


def test_logits_with_norm_and_strides():
    B, K, V, group = 6, 1280, 301, 64
    q = weight(V, K, group, False, seed=9)
    big = torch.full((B, K + 40), float("nan"), dtype=torch.bfloat16, device="cuda")
    big[:, :K] = 3.0 * torch.randn(B, K, device="cuda", generator=gen(1))
    nw = (1.0 + 0.2 * torch.randn(K, device="cuda", generator=gen(2))).to(torch.bfloat16)
    x = big[:, :K]
    ref = H.rms_norm(x.float().cpu().numpy(), nw.float().cpu().numpy(), 1e-6)
    xn = torch.from_numpy(ref).cuda().to(torch.bfloat16)
    got = ops.head_logits_q4(x, q, norm_weight=nw)
    check_logits(xn, q, got, "norm")
    assert torch.equal(got, ops.head_logits_q4(xn, q))
    # strided weights and logits through the C entry
    lib, s = N.lib(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    words = torch.full((V, K // 8 + 12), -1, dtype=torch.int32, device="cuda")
    sc = torch.full((V, K // group + 3), float("nan"), dtype=torch.bfloat16, device="cuda")
    bi = sc.clone()
    words[:, :K // 8], sc[:, :K // group], bi[:, :K // group] = q.words, q.scales, q.biases
    buf = torch.full((B, V + 5), 7.0, device="cuda")
    ws = torch.empty(lib.strim_head_logits_packed_workspace(B, K), dtype=torch.uint8, device="cuda")

    def p(t):
        return ctypes.c_void_p(t.data_ptr())

    rc = lib.strim_head_logits_packed(s, p(xn), K, B, K, None, 1e-6, None, p(words), K // 8 + 12,
                                      p(sc), p(bi), K // group + 3, group, V, p(ws), ws.numel(),
                                      p(buf), N.DTYPE_F32, V + 5)
    assert rc == N.OK
    torch.cuda.synchronize()
    assert torch.equal(buf[:, :V], ops.head_logits_q4(xn, q, out_dtype=torch.float32))
    assert bool((buf[:, V:] == 7.0).all())


def test_a_bad_row_stays_in_its_row():
    """A NaN in a hidden row, or in a weight row's scales, reaches that row's logits alone."""
    for B in (3, 12, 40):
        q = weight(90, 512, 64, False, seed=3)
        x = torch.randn(B, 512, device="cuda", generator=gen(3)).to(torch.bfloat16)
        ref = ops.head_logits_q4(x, q)
        x[1, 100] = float("nan")
        q.scales[17, 2] = float("nan")
        got = ops.head_logits_q4(x, q)
        assert bool(got[1].isnan().all()) and bool(got[:, 17].isnan().all())
        keep = torch.ones(B, 90, dtype=torch.bool, device="cuda")
        keep[1], keep[:, 17] = False, False
        assert torch.equal(got[keep], ref[keep])


def test_logits_in_a_graph_then_sampled():
    q = weight(2000, 512, 64, False, seed=5)
    x = torch.randn(4, 512, device="cuda", generator=gen(5)).to(torch.bfloat16)
    out = torch.empty(4, 2000, dtype=torch.bfloat16, device="cuda")
    ops.head_logits_q4(x, q, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.head_logits_q4(x, q, out=out)
        ids = ops.draft_argmax(out)
    for seed in (6, 7, 8):
        x.copy_(torch.randn(4, 512, device="cuda", generator=gen(seed)))
        graph.replay()
        torch.cuda.synchronize()
        ref = ops.head_logits_q4(x, q)
        assert torch.equal(out, ref)
        assert torch.equal(ids.long(), ref.float().argmax(1))


def test_refusals():
    q = weight(20, 256, 64, False, seed=1)
    x = torch.randn(2, 256, device="cuda").to(torch.bfloat16)
    w = torch.randn(20, 256, device="cuda")
    with pytest.raises(TypeError):
        ops.head_logits_q4(x.float(), q)
    with pytest.raises(ValueError):
        ops.head_logits_q4(x[:, :128], q)
    with pytest.raises(ValueError):
        ops.head_logits_q4(x.cpu(), q)
    with pytest.raises(TypeError):
        ops.head_logits_q4(x, q, out_dtype=torch.float16)
    with pytest.raises(ValueError):
        ops.head_logits_q4(x, q, out=torch.empty(2, 19, device="cuda"))
    with pytest.raises(ValueError):
        ops.Q4Weight(q.words, q.scales, q.biases, 32)
    with pytest.raises(ValueError):
        ops.Q4Weight(q.words.long(), q.scales)
    with pytest.raises(ValueError):
        ops.Q4Weight(q.words, q.scales.float(), None)
    with pytest.raises(ValueError):
        ops.q4_pack(w, 48)
    with pytest.raises(ValueError):
        ops.q4_pack(w[:, :100], 64)
    with pytest.raises(TypeError):
        ops.q4_pack(w.half())
    lib, s = N.lib(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    out = torch.empty(2, 20, device="cuda")
    need = lib.strim_head_logits_packed_workspace(2, 256)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")

    def p(t):
        return ctypes.c_void_p(t.data_ptr())

    def call(**kw):
        a = dict(hs=256, B=2, K=256, nw=None, xn=None, wst=32, ss=4, g=64, V=20, ws=p(ws), wb=need,
                 dt=N.DTYPE_F32, os=20)
        a.update(kw)
        return lib.strim_head_logits_packed(s, p(x), a["hs"], a["B"], a["K"], a["nw"], 1e-6, a["xn"],
                                            p(q.words), a["wst"], p(q.scales), p(q.biases), a["ss"],
                                            a["g"], a["V"], a["ws"], a["wb"], p(out), a["dt"], a["os"])

    assert call() == N.OK
    assert call(B=0) == N.EINVAL
    assert call(K=224) == N.EINVAL
    assert call(g=16) == N.EINVAL
    assert call(hs=248) == N.EINVAL
    assert call(wst=31) == N.EINVAL
    assert call(ss=3) == N.EINVAL
    assert call(os=19) == N.EINVAL
    assert call(dt=7) == N.EINVAL
    assert call(nw=p(x)) == N.EINVAL
    assert call(ws=None) == N.EINVAL
    assert call(wb=need - 1) == N.ECAPACITY
    torch.cuda.synchronize()


@pytest.mark.parametrize("symmetric", [False, True])
def test_pack_scales_near_the_ends_of_the_range(symmetric):
    """Groups whose scale is subnormal, huge, or exactly between two codes everywhere: the codes
    are those of the correctly rounded quotient."""
    K, G = 256, 64
    w = torch.randn(40, K, device="cuda", generator=gen(6))
    w *= torch.exp2(torch.linspace(-140, 120, 40, device="cuda"))[:, None]
    w[3] = (torch.arange(K, device="cuda") % 31) * 0.5  # halves of a step
    w[3, ::G] = 0.0
    w[3, 1::G] = 15.0
    w[3, 2::G] = -7.0 if symmetric else 0.0
    q = ops.q4_pack(w, G, symmetric)
    d = w.reshape(40, -1, G)
    s = q.scales.float()[..., None]
    if symmetric:
        ref = torch.where(s > 0, d / s, 0.0).round() + 8
    else:
        ref = torch.where(s > 0, (d - q.biases.float()[..., None]) / s, 0.0).round()
    assert torch.equal(codes(q), ref.clamp(0, 15).double())


def test_offsets_past_32_bits():
    """Words of more than 2^31 bytes: the last rows' logits, read back values and packing."""
    V, K, G = 430_000, 10_240, 128
    print("[q4] 2^31 bytes", flush=True)
    q = weight(V, K, G, False, seed=77)
    tail = ops.Q4Weight(q.words[-300:].contiguous(), q.scales[-300:].contiguous(),
                        q.biases[-300:].contiguous(), G)
    for B in (2, 20):
        x = torch.randn(B, K, device="cuda", generator=gen(B)).to(torch.bfloat16)
        got = ops.head_logits_q4(x, q)
        check_logits(x, tail, got[:, -300:], f"B={B}")
    v = ops.q4_unpack(q)
    assert torch.equal(v[-300:], ops.q4_unpack(tail))
    p = ops.q4_pack(v, G)
    t = ops.q4_pack(v[-300:].contiguous(), G)
    assert torch.equal(p.words[-300:], t.words) and torch.equal(p.scales[-300:], t.scales)


@pytest.mark.parametrize("B,K,V,G,sym", [
    (9, 2080, 1, 32, False), (16, 5152, 300, 32, True), (16, 5120, 4099, 64, False),
    (33, 2112, 16_001, 64, True), (64, 8192, 4111, 128, False), (70, 5120, 2049, 64, False),
    (130, 2048, 70, 128, True)])
def test_few_weight_rows(B, K, V, G, sym):
    """Less than a round of row tiles: K in parts, their sums joined."""
    print(f"[q4] parts of K: B={B} V={V} K={K} G={G}", flush=True)
    q = weight(V, K, G, sym, seed=B + K)
    x = torch.randn(B, K, device="cuda", generator=gen(V)).to(torch.bfloat16)
    check_logits(x, q, ops.head_logits_q4(x, q), "bf16")
    y = ops.head_logits_q4(x, q, out_dtype=torch.float32)
    check_logits(x, q, y, "f32")
    assert torch.equal(y, ops.head_logits_q4(x, q, out_dtype=torch.float32))


@pytest.mark.parametrize("B,K,V,G", [
    (33, 1024, 34_001, 64), (40, 544, 60_001, 32), (64, 640, 98_003, 64), (64, 1024, 130_007, 128),
    (50, 1056, 160_001, 32), (64, 1152, 163_839, 128), (17, 640, 98_003, 64), (32, 544, 131_001, 32),
    (32, 1152, 163_841, 128)])
def test_several_tiles_a_wave(B, K, V, G):
    """Rounds of two to five row tiles a wave, full and not."""
    print(f"[q4] rounds: B={B} V={V} K={K} G={G}", flush=True)
    q = weight(V, K, G, False, seed=B + K)
    x = torch.randn(B, K, device="cuda", generator=gen(V)).to(torch.bfloat16)
    check_logits(x, q, ops.head_logits_q4(x, q, out_dtype=torch.float32), "f32")


def test_norm_of_more_rows_than_a_launch_has():
    """More rows to normalise than workgroups of 1,024 threads in a launch. The rows repeat 64."""
    R, K, V, M = 64, 32, 5, 1 << 16
    B = R * M + 1
    print(f"[q4] norm B={B}", flush=True)
    q = weight(V, K, 32, False, seed=8)
    x = torch.randn(R, K, device="cuda", generator=gen(8)).to(torch.bfloat16)
    nw = torch.ones(K, dtype=torch.bfloat16, device="cuda")
    ref = ops.head_logits_q4(x, q, nw)
    got = ops.head_logits_q4(torch.cat([x.repeat(M, 1), x[:1]]), q, nw)
    assert bool((got[:-1].view(M, R, V) == ref).all()) and torch.equal(got[-1], ref[0])


@pytest.mark.parametrize("B", [2, 8, 16, 64])
def test_an_infinity_stays_in_its_row(B):
    """A hidden row that holds an infinity has no finite logit; the other rows keep their bits."""
    q = weight(300, 512, 64, True, seed=9)
    x = torch.randn(B, 512, device="cuda", generator=gen(9)).to(torch.bfloat16)
    ref = ops.head_logits_q4(x, q)
    x[B // 2, 77] = float("-inf")
    got = ops.head_logits_q4(x, q)
    assert not bool(got[B // 2].isfinite().any())
    keep = torch.arange(B, device="cuda") != B // 2
    assert torch.equal(got[keep], ref[keep])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("symmetric", [False, True])
def test_pack_scales_are_the_products(symmetric, dtype):
    """A stored scale is the float32 product of the group's width and the float32 number next to 1 / 15
    (1 / 7), rounded to bf16, also where the quotient is exactly between two bf16 numbers; its codes
    are the nearest ones for that scale."""
    if symmetric and dtype == torch.bfloat16:
        n = torch.arange(1, 256, device="cuda").double().repeat(2)  # (no 8-bit number is 7 times such a one)
    else:
        n = torch.arange(257, 512, 2, device="cuda").double() * (7 if symmetric else 15)
    n = torch.cat([n * 2.0 ** e for e in (-9, -1, 6)])
    V, G = n.numel(), 64
    u = torch.rand(V, G, device="cuda", dtype=torch.float64, generator=gen(12))
    if symmetric:
        w = (2 * u - 1) * n[:, None]
        w[:, 5], w[:, 9] = n, -n
    else:
        lo = -torch.remainder(n, 32 * 2.0 ** torch.floor(torch.log2(n) - 12))  # n's bits past the first eight
        w = lo[:, None] + u * n[:, None]
        w[:, 5], w[:, 9] = lo, n + lo
    w = w.to(dtype)
    q = ops.q4_pack(w, G, symmetric)
    d = w.double()
    hi, lo = d.amax(1), d.amin(1)
    assert torch.equal(hi if symmetric else hi - lo, n)
    s = (n.float() * torch.full_like(n, 1 / (7 if symmetric else 15), dtype=torch.float32)).to(torch.bfloat16)
    assert torch.equal(q.scales[:, 0], s)
    base = torch.zeros_like(lo) if symmetric else lo.to(torch.bfloat16).double()
    if not symmetric:
        assert torch.equal(q.biases[:, 0].double(), base)
    want = ((d.float() - base.float()[:, None]) / s.float()[:, None]).round() + (8 if symmetric else 0)
    assert torch.equal(codes(q)[:, 0], want.clamp(0, 15).double())
