"""Token scores (strim_token_scores, strim_token_scores_grad and their differentiable form) against the
formulas in float64, and against differences.

The bounds follow from float32 arithmetic. With d = x - max, D = sum p |d| / T, D2 = sum p (d / T)^2:
  a term exp(d / T) is off by (|d| / T) 2^-23 (its exponent's two roundings) and 2^-22 (the exponential),
  a sum of V terms by one rounding an addition, of which a chain has V / 256 and 40 for the merges:
  c = (V / 256 + 40) 2^-24;
  lse, a log-probability: e = c + 2^-22 (8 + D) and 2^-22 of its terms |x - max| / T and |lse|;
  the entropy: e + (c + 2^-22 8) D + 2^-22 (D2 + D);
  a gradient: its p is off by e + 2^-21 (1 + |lse| + |x| / T), its log p + H by both values' errors; one
  rounding to its type."""
import ctypes

import pytest
import torch

from strim_amd import _native as N
from strim_amd import loss as L
from strim_amd import ops

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def logits(R, V, dtype, seed, peaks=4):
    g = gen(seed)
    x = 2.0 * torch.randn(R, V, device="cuda", generator=g)
    at = torch.randint(0, V, (R, peaks), device="cuda", generator=g)
    x.scatter_(1, at, 4.0 + 8.0 * torch.rand(R, peaks, device="cuda", generator=g))
    return x.to(dtype)


def pitched(t, pad, shift=0):
    """The same rows `pad` elements further apart, `shift` elements into their memory, NaN between."""
    R, V = t.shape
    buf = torch.full((R * (V + pad) + shift,), float("nan"), dtype=t.dtype, device=t.device)
    out = buf[shift:].view(R, V + pad)[:, :V]
    out.copy_(t)
    return out


def words_of(allowed):
    return ops.pack_mask(allowed)


def within(got, ref, tol, what):
    got, ref = got.double(), ref.double()
    same = (got == ref) | (got.isnan() & ref.isnan())
    err = torch.where(same, 0.0, (got - ref).abs())
    bad = ~(err <= tol)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} past the bound, worst "
                                 f"{float((err / tol).nan_to_num(1e9).max()):.3g} of it")


class Exact:
    def __init__(self, x, T=1.0, allowed=None):
        self.x = x.double() if allowed is None else torch.where(allowed, x.double(), float("-inf"))
        self.T, self.V = T, x.shape[1]
        top = self.x.amax(1, keepdim=True)
        self.z = self.x / T
        self.lse = torch.logsumexp(self.z, 1)
        self.lp = torch.where(self.z == float("-inf"), float("-inf"), self.z - self.lse[:, None])
        p = torch.exp(self.lp)
        self.p = p
        self.H = -(p * self.lp.nan_to_num(neginf=0.0)).sum(1)
        d = ((self.x - top).abs() / T).nan_to_num(posinf=0.0)
        D, D2 = (p * d).sum(1), (p * d * d).sum(1)
        c = (self.V / 256 + 40) * 2.0 ** -24
        self.e = c + 2.0 ** -22 * (8 + D)
        self.tol_lse = self.e + 2.0 ** -22 * self.lse.abs().nan_to_num(posinf=0.0)
        self.tol_H = self.e + (c + 2.0 ** -19) * D + 2.0 ** -22 * (D2 + D)
        self.d = d

    def tol_lp(self, at):
        return self.e[:, None] + 2.0 ** -22 * (self.d.gather(1, at) + self.lse.abs()[:, None].nan_to_num(posinf=0.0))

    def top(self, n):
        x, ids = torch.sort(self.x, dim=1, descending=True, stable=True)
        if n > self.V:
            pad = torch.full((x.shape[0], n - self.V), float("-inf"), dtype=x.dtype, device=x.device)
            x, ids = torch.cat([x, pad], 1), torch.cat([ids, torch.zeros_like(pad, dtype=ids.dtype)], 1)
        x, ids = x[:, :n], ids[:, :n]
        lp = self.lp.gather(1, ids)
        none = x == float("-inf")
        return (torch.where(none, -1, ids).to(torch.int32), torch.where(none, float("-inf"), lp),
                self.tol_lp(ids))

    def grad(self, tokens, g, gh, gl, eps):
        """(gradient, bound) for tokens [R, S] all inside the vocabulary."""
        g, gh, gl = (0.0 if t is None else t.double() for t in (g, gh, gl))
        R = self.x.shape[0]
        G = g.sum(1) if isinstance(g, torch.Tensor) else torch.zeros(R, device="cuda").double()
        gh = torch.zeros_like(G) + gh
        gl = torch.zeros_like(G) + gl
        lp = self.lp.nan_to_num(neginf=0.0)
        d = -self.p * ((G - gl)[:, None] + gh[:, None] * (lp + self.H[:, None]))
        mag = self.p * ((G.abs() + gl.abs())[:, None] + gh.abs()[:, None] * (lp.abs() + self.H[:, None]))
        rel = self.e[:, None] + 2.0 ** -21 * (1 + self.lse.abs()[:, None] + self.z.abs().nan_to_num(posinf=0.0))
        tol = mag * rel + self.p * gh.abs()[:, None] * (self.tol_H[:, None] + rel)
        if isinstance(g, torch.Tensor):
            inside = (self.x > float("-inf")).gather(1, tokens)
            d.scatter_add_(1, tokens, torch.where(inside, g, 0.0))
            tol.scatter_add_(1, tokens, 2.0 ** -22 * g.abs())
        d = torch.where(self.x > float("-inf"), d, 0.0) / self.T
        tol = tol / self.T
        return d, tol + (d.abs() + tol) * eps + 1e-37


def check(x, tokens, top, T=1.0, allowed=None, label=""):
    R, V = x.shape
    E = Exact(x, T, allowed)
    out = ops.token_scores(x, tokens, top, T, None if allowed is None else words_of(allowed))
    assert bool((out.status == 0).all()), out.status
    within(out.lse, E.lse, E.tol_lse, f"{label} lse")
    within(out.entropy, E.H, E.tol_H, f"{label} entropy")
    t = tokens.long().reshape(R, -1)
    within(out.logprobs.reshape(R, -1), E.lp.gather(1, t), E.tol_lp(t), f"{label} log-probabilities")
    assert out.logprobs.shape == tokens.shape
    if top:
        ids, lp, tol = E.top(top)
        assert torch.equal(out.top_ids, ids), f"{label}: {int((out.top_ids != ids).sum())} ids"
        within(out.top_logprobs, lp, tol, f"{label} alternatives")
    # without the alternatives, and without tokens: the same bits
    again = ops.token_scores(x, None, 0, T, None if allowed is None else words_of(allowed))
    assert again.logprobs is None and again.top_ids is None
    within(again.lse, E.lse, E.tol_lse, f"{label} lse alone")
    within(again.entropy, E.H, E.tol_H, f"{label} entropy alone")
    return out, E


SIZES = [(1, 1, 1), (1, 5, 8), (2, 8, 3), (3, 257, 20), (5, 4095, 20), (4, 4097, 1), (2, 8192, 128),
         (7, 20_001, 64), (64, 9_000, 5), (300, 1_500, 100), (1, 151_936, 20), (9, 151_936, 128),
         (3, 248_320, 20), (600, 32_768, 64), (1100, 10_007, 20)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,V,top", SIZES)
def test_scores(R, V, top, dtype):
    print(f"[scores] R={R} V={V} top={top} {dtype}", flush=True)
    x = logits(R, V, dtype, seed=R + V)
    t = torch.randint(0, V, (R,), device="cuda", generator=gen(1)).to(torch.int32)
    check(x, t, top, label=f"R={R} V={V}")


@pytest.mark.parametrize("R,V,top,T,S", [(3, 700, 20, 0.7, 2), (5, 33, 40, 2.0, 1), (64, 5_003, 8, 0.8, 4),
                                         (40, 100_003, 30, 1.3, 128), (513, 4_100, 20, 0.5, 1)])
def test_masks_temperature_and_several_tokens(R, V, top, T, S):
    """Masks that allow most ids, few, one run of neighbours, or a single one; log-probabilities of
    several tokens, also the same one twice and forbidden ones."""
    print(f"[scores] masked R={R} V={V}", flush=True)
    g = gen(V)
    x = logits(R, V, torch.bfloat16, seed=V)
    keep = torch.tensor([0.95, 0.02, 0.0, 0.0], device="cuda")[torch.arange(R, device="cuda") % 4]
    allowed = torch.rand(R, V, device="cuda", generator=g) < keep[:, None]
    first = torch.randint(0, V, (R, 1), device="cuda", generator=g)
    at = torch.arange(V, device="cuda")
    allowed |= (at >= first) & (at <= first + torch.where(torch.arange(R, device="cuda") % 4 == 2, 30, 0)[:, None])
    t = torch.randint(0, V, (R, S), device="cuda", generator=g).to(torch.int32)
    t[:, -1] = first[:, 0]
    t[:, 0] = t[:, -1]
    check(x, t if S > 1 else t[:, 0].contiguous(), top, T, allowed, "masked")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pad,shift", [(3, 0), (8, 8), (1, 1), (0, 5)])
def test_strides_and_unaligned_rows(pad, shift, dtype):
    for R, V in ((5, 1_003), (3, 9_001), (130, 5_000)):
        print(f"[scores] pitch +{pad} shift {shift} R={R} V={V} {dtype}", flush=True)
        x = pitched(logits(R, V, dtype, seed=7), pad, shift)
        t = torch.randint(0, V, (R,), device="cuda", generator=gen(2)).to(torch.int32)
        out, E = check(x, t, 20, label="pitched")
        gl, gh = torch.randn(R, device="cuda", generator=gen(3)), torch.randn(R, device="cuda", generator=gen(4))
        into = pitched(torch.zeros_like(x), pad + 2, shift)
        guard = into.as_strided((R, pad + 2), (V + pad + 2, 1), into.storage_offset() + V) if R > 1 else None
        d = ops.token_scores_grad(x, t, out.lse, out.entropy, gl, gh, out=into)
        assert d is into
        ref, tol = E.grad(t.long()[:, None], gl[:, None], gh, None, torch.finfo(dtype).eps / 2)
        within(d, ref, tol, "pitched gradient")
        if guard is not None:  # what lies between the rows stays
            assert bool(guard[:-1].isnan().all())


def rows_of_every_kind(V, dtype):
    """Rows whose alternatives are hard to pick: by name."""
    dev, ninf = "cuda", float("-inf")
    base = torch.randn(V, device=dev, generator=gen(9))
    rows = {
        "flat": torch.zeros(V), "flat but one": torch.zeros(V).index_fill(0, torch.tensor([V // 2]), 3.0),
        "ascending": torch.linspace(-20, 20, V), "descending": torch.linspace(20, -20, V),
        "quantised": (base * 2).round().cpu(), "signed zeros": torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0),
        "few above the lowest value": torch.full((V,), torch.finfo(dtype).min).index_fill(
            0, torch.tensor([1, V // 3, V - 1]), 1.0),
        "few finite": torch.full((V,), ninf).index_fill(0, torch.tensor([0, V // 2, V - 1]), -1.0),
        "one finite": torch.full((V,), ninf).index_fill(0, torch.tensor([V - 2]), 5.0),
        "a run of large ones": torch.where((torch.arange(V) // 64) % 50 == 3, 10.0 + base.cpu(), base.cpu()),
        "one lane's": torch.where(torch.arange(V) % 2048 < 8, 9.0 + base.cpu(), base.cpu()),
        "far below zero": base.cpu() - 3e4, "wide": base.cpu() * 1e4, "nearly certain": base.cpu().index_fill(
            0, torch.tensor([V // 4]), 60.0),
        "ends": base.cpu().index_fill(0, torch.tensor([0, V - 1]), 12.0),
    }
    return list(rows), torch.stack([r.to(dev) for r in rows.values()]).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,top,copies", [(40, 20, 1), (4_099, 128, 1), (30_011, 100, 1), (20_480, 64, 60),
                                          (151_936, 128, 1)])
def test_rows_of_every_kind(V, top, copies, dtype):
    names, x = rows_of_every_kind(V, dtype)
    print(f"[scores] kinds V={V} {dtype}: {names}", flush=True)
    x = x.repeat(copies, 1)
    check(x, torch.full((x.shape[0],), V - 1, dtype=torch.int32, device="cuda"), top, label=f"V={V}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,top,copies", [(33_000, 5, 1), (151_936, 128, 1), (20_480, 128, 110), (70_001, 1, 40)])
def test_rows_whose_waves_differ(V, top, copies, dtype):
    """Plateaus and runs that fill some waves' lists and not others', ties across them."""
    at = torch.arange(V)
    part = at // 512 % 4  # (which wave of a workgroup meets a token)
    base = torch.randn(V, generator=torch.Generator().manual_seed(3))
    rows = [(at // 1500).float() / 8, -(at // 1500).float() / 8, torch.where(part == 0, at.float() / V * 40, base),
            torch.where(part == 2, (at // 4096).float(), base.round()), torch.where(part == 1, 3.0, 2.5 + 0 * base),
            torch.where(part == 3, base.round() + at // 16384, base.round() + (at // 16384).flip(0)),
            torch.where(at // 2048 % 9 == 4, 7.0, base), (base * 4).round() / 4 + (at // 8192) * 0.25]
    x = torch.stack(rows).to("cuda", dtype).repeat(copies, 1)
    print(f"[scores] waves V={V} top={top} {dtype}", flush=True)
    check(x, torch.full((x.shape[0],), 0, dtype=torch.int32, device="cuda"), top, label=f"V={V}")


def test_statuses():
    """Empty rows, NaN and infinities in allowed and forbidden places, unknown and ignored tokens; what
    the others in the batch give is not touched."""
    V, nan, inf = 5_000, float("nan"), float("inf")
    for dtype in (torch.bfloat16, torch.float32):
        x = logits(8, V, dtype, seed=4)
        clean = x.clone()
        allowed = torch.ones(8, V, dtype=torch.bool, device="cuda")
        allowed[0] = False                       # nothing allowed
        x[1] = -inf                              # nothing finite
        x[2, 4_000] = nan                        # NaN allowed
        x[3, 17], x[3, 4_097] = inf, nan         # both forbidden
        allowed[3, 17] = allowed[3, 4_097] = False
        x[4, 4_999] = inf                        # +inf allowed
        x[5, :4_990] = -inf                      # ten left
        t = torch.tensor([3, 3, 3, 3, 3, 4_995, 5_000, -100], dtype=torch.int32, device="cuda")
        out = ops.token_scores(x, t, 20, mask=words_of(allowed))
        st = [N.EEMPTY, N.EEMPTY, N.ENONFINITE, N.OK, N.ENONFINITE, N.OK, N.EINVAL, N.OK]
        assert out.status.tolist() == st
        assert out.lse[:2].tolist() == [-inf, -inf] and out.entropy[:2].tolist() == [0.0, 0.0]
        assert out.logprobs[:2].tolist() == [-inf, -inf]
        assert bool((out.top_ids[:2] == -1).all()) and bool((out.top_logprobs[:2] == -inf).all())
        for r in (2, 4):
            assert bool(out.lse[r].isnan()) and bool(out.entropy[r].isnan()) and bool(out.logprobs[r].isnan())
            assert bool((out.top_ids[r] == -1).all()) and bool(out.top_logprobs[r].isnan().all())
        assert out.logprobs[6:].tolist() == [0.0, 0.0]
        good = [3, 5, 6, 7]
        E = Exact(torch.where(allowed, x, clean)[good], 1.0, allowed[good])
        within(out.lse[good], E.lse, E.tol_lse, "lse")
        ids, lp, tol = E.top(20)
        assert torch.equal(out.top_ids[good], ids)
        within(out.top_logprobs[good], lp, tol, "alternatives")
        # another ignored id, one of the vocabulary
        other = ops.token_scores(x, t, 0, mask=words_of(allowed), ignore_index=3)
        assert other.logprobs[3].item() == 0.0 and other.status.tolist() == st[:7] + [N.EINVAL]
        # gradients: empty rows none, unknown and ignored tokens none, NaN where allowed
        g = torch.ones(8, device="cuda")
        d = ops.token_scores_grad(x, t, out.lse, out.entropy, g, g, mask=words_of(allowed))
        assert bool((d[:2] == 0).all()) and bool(d[2].isnan().all()) and bool(d[4].isnan().all())
        assert bool((d[~allowed] == 0).all())
        only = ops.token_scores_grad(x, t, out.lse, None, g, mask=words_of(allowed))
        assert bool((only[6:] == 0).all())
        assert d[3].isfinite().all() and d[5].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,V,S,T", [(1, 7, 1, 1.0), (4, 1_000, 3, 0.7), (33, 9_001, 1, 2.0), (2, 151_936, 128, 1.0),
                                     (700, 2_050, 2, 1.0)])
def test_gradients(R, V, S, T, dtype):
    print(f"[scores] gradients R={R} V={V} S={S} {dtype}", flush=True)
    x = logits(R, V, dtype, seed=R)
    t = torch.randint(0, V, (R, S), device="cuda", generator=gen(5)).to(torch.int32)
    if S > 1:
        t[:, 1] = t[:, 0]  # the same token twice
    out = ops.token_scores(x, t, 0, T)
    E = Exact(x, T)
    g = torch.randn(R, S, device="cuda", generator=gen(6))
    gh, gl = (torch.randn(R, device="cuda", generator=gen(s)) for s in (7, 8))
    eps = torch.finfo(dtype).eps / 2
    for args in ((g, gh, gl), (g, None, None), (None, gh, None), (None, None, gl), (g, gh, None)):
        d = ops.token_scores_grad(x, t, out.lse, out.entropy, *args, temperature=T)
        within(d, *E.grad(t.long(), *args, eps), f"{[a is not None for a in args]}")
    # into the logits themselves
    y = x.clone()
    ops.token_scores_grad(y, t, out.lse, out.entropy, g, gh, None, temperature=T, out=y)
    assert torch.equal(y, d)
    assert bool((ops.token_scores_grad(x, t, out.lse) == 0).all())


def test_masked_gradients():
    R, V, T = 24, 6_001, 0.8
    x = logits(R, V, torch.float32, seed=12)
    allowed = torch.rand(R, V, device="cuda", generator=gen(13)) < 0.3
    t = torch.randint(0, V, (R, 2), device="cuda", generator=gen(14)).to(torch.int32)
    allowed[:, 5] = True
    allowed.scatter_(1, t[:, :1].long(), True)
    x[~allowed] = float("nan")
    out = ops.token_scores(x, t, 0, T, words_of(allowed))
    E = Exact(torch.where(allowed, x, 0.0), T, allowed)
    g, gh = torch.randn(R, 2, device="cuda", generator=gen(15)), torch.randn(R, device="cuda", generator=gen(16))
    d = ops.token_scores_grad(x, t, out.lse, out.entropy, g, gh, temperature=T, mask=words_of(allowed))
    within(d, *E.grad(t.long(), g, gh, None, 2.0 ** -24), "masked")


def test_differences():
    """Gradients along directions against differences of the scores: steps of 1/16 on a grid of 1/8, exact
    in float32. The third derivative of an entropy or a log-probability along a step h of logits is below
    8 (1 + H) h^3; the values are off by 1e-5 at most."""
    R, V = 16, 900
    x = (torch.randn(R, V, device="cuda", generator=gen(20)) * 8).round() / 8
    t = torch.randint(0, V, (R,), device="cuda", generator=gen(21)).to(torch.int32)
    out = ops.token_scores(x, t)
    one, none = torch.ones(R, device="cuda"), None
    grads = [ops.token_scores_grad(x, t, out.lse, out.entropy, *a) for a in
             ((one, none, none), (none, one, none), (none, none, one))]
    for s in range(6):
        d = torch.where(torch.rand(R, V, device="cuda", generator=gen(30 + s)) < 0.5, -1.0, 1.0)
        up, dn = ops.token_scores(x + d / 16, t), ops.token_scores(x - d / 16, t)
        for grad, a, b in zip(grads, up[:3], dn[:3]):
            diff, lin = (a - b).double() * 8, (grad.double() * d).sum(1)
            tol = 16e-5 + 8 * 8 * (1 + out.entropy.double()) / 16 ** 3 / 6
            assert bool(((diff - lin).abs() <= tol).all()), float(((diff - lin).abs() - tol).max())


def test_past_32_bits():
    """More than 2^31 elements, and 2^32 bytes, in both tensors."""
    R, V = 14_200, 151_936
    x = torch.zeros(R, V, dtype=torch.bfloat16, device="cuda")
    last = [0, 7_000, R - 1]
    x[last] = logits(3, V, torch.bfloat16, seed=3)
    t = torch.full((R,), V - 1, dtype=torch.int32, device="cuda")
    out = ops.token_scores(x, t, 4)
    E = Exact(x[last])
    within(out.lse[last], E.lse, E.tol_lse, "lse")
    ids, _, _ = E.top(4)
    assert torch.equal(out.top_ids[last], ids)
    flat = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
    assert bool((out.top_ids[1:7_000] == flat).all())
    g = torch.ones(R, device="cuda")
    d = ops.token_scores_grad(x, t, out.lse, out.entropy, g, g, out=x)
    within(d[last], *E.grad(t[last].long()[:, None], g[:3, None], g[:3], None, 2.0 ** -8), "gradient")


def test_autograd():
    """Shapes, token types, gradients through every output that has one, unused outputs, a broadcast
    gradient, a transposed batch, second derivatives refused."""
    x = logits(60, 500, torch.float32, seed=31).reshape(3, 20, 500)
    t = torch.randint(0, 500, (3, 20), device="cuda", generator=gen(32))
    leaf = x.clone().requires_grad_()
    out = L.token_scores(leaf, t, top=3, temperature=0.9)
    assert out.logprobs.shape == (3, 20) and out.top_ids.shape == (3, 20, 3)
    assert not out.top_logprobs.requires_grad and not out.status.requires_grad
    (out.logprobs.mean() - 0.01 * out.entropy.sum()).backward()
    E = Exact(x.reshape(60, 500), 0.9)
    one = torch.ones(60, device="cuda")
    within(leaf.grad.reshape(60, 500), *E.grad(t.reshape(60, 1), one[:, None] / 60, -0.01 * one, None, 2.0 ** -24),
           "both")
    leaf.grad = None
    L.token_scores(leaf, None, temperature=0.9).lse.sum().backward()
    within(leaf.grad.reshape(60, 500), *E.grad(None, None, None, one, 2.0 ** -24), "lse")
    # several tokens a row, int64 ids past 32 bits, a view whose rows are not contiguous
    many = torch.stack([t, t, torch.full_like(t, 2 ** 40)], 2)
    wide = x.transpose(1, 2).contiguous().transpose(1, 2).detach().requires_grad_()
    out = L.token_scores(wide, many)
    assert out.logprobs.shape == (3, 20, 3) and bool((out.logprobs[..., 2] == 0).all())
    assert bool((out.status == N.EINVAL).all())
    out.logprobs.sum().backward()
    E = Exact(x.reshape(60, 500))
    within(wide.grad.reshape(60, 500), *E.grad(t.reshape(60, 1), 2 * one[:, None], None, None, 2.0 ** -24), "wide")
    (d,) = torch.autograd.grad(L.token_scores(leaf, t).entropy.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        d.square().sum().backward()


def test_repeatable_streams_and_graphs():
    """The same bits again, on another stream and from a graph replayed with other inputs between the
    program's own work; two graphs over one workspace."""
    R, V = 40, 50_003
    x, x2 = (logits(R, V, torch.bfloat16, seed=s) for s in (41, 42))
    t = torch.randint(0, V, (R,), device="cuda", generator=gen(43)).to(torch.int32)
    g = torch.randn(R, device="cuda", generator=gen(44))
    ws = torch.empty(max(16, ops.token_scores_workspace(R, V, 20)), dtype=torch.uint8, device="cuda")

    def run(workspace=None):
        out = ops.token_scores(x, t, 20, workspace=workspace)
        return [*out, ops.token_scores_grad(x, t, out.lse, out.entropy, g, g)]

    ref = run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    out = ops.token_scores(x, t, 20, stream=stream)
    d = ops.token_scores_grad(x, t, out.lse, out.entropy, g, g, stream=stream)
    torch.cuda.current_stream().wait_stream(stream)
    for a, b in zip([*out, d], ref):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = run(ws)
        graphs.append((graph, res))
    keep = x.clone()
    for src in (x2, keep, x2):
        x.copy_(src)
        ref = run()
        for graph, res in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, res in graphs:
            for a, b in zip(res, ref):
                assert torch.equal(a, b)


def test_no_rows():
    x = torch.empty(0, 100, dtype=torch.bfloat16, device="cuda")
    out = ops.token_scores(x, torch.empty(0, dtype=torch.int32, device="cuda"), 5)
    assert out.lse.shape == (0,) and out.top_ids.shape == (0, 5)
    assert ops.token_scores_grad(x, None, out.lse).shape == (0, 100)


def test_refusals():
    x = logits(4, 100, torch.bfloat16, seed=1)
    t = torch.zeros(4, dtype=torch.int32, device="cuda")
    out = ops.token_scores(x, t)
    bad = [lambda: ops.token_scores(x.T, t), lambda: ops.token_scores(x, t[:3]),
           lambda: ops.token_scores(x, t.long()), lambda: ops.token_scores(x, t, -1),
           lambda: ops.token_scores(x, t, 129), lambda: ops.token_scores(x, t, temperature=0.0),
           lambda: ops.token_scores(x, t, temperature=float("nan")),
           lambda: ops.token_scores(x, t, mask=torch.zeros(4, 3, dtype=torch.int32, device="cuda")),
           lambda: ops.token_scores(x, t, mask=torch.zeros(3, 4, dtype=torch.int32, device="cuda")),
           lambda: ops.token_scores(x, t.cpu()), lambda: ops.token_scores(x.cpu(), t),
           lambda: ops.token_scores(x, t.expand(130, 4).T.contiguous()),
           lambda: ops.token_scores(x, t, ignore_index=2 ** 31),
           lambda: ops.token_scores(x.expand(4, 4, 100), t), lambda: ops.token_scores(x[:1].expand(4, 100), t),
           lambda: ops.token_scores_grad(x, t, out.lse[:3]),
           lambda: ops.token_scores_grad(x, t, out.lse, None, None, out.lse),
           lambda: ops.token_scores_grad(x, None, out.lse, None, out.lse),
           lambda: ops.token_scores_grad(x, t, out.lse, out=x.float())]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        ops.token_scores(x.half(), t)
    need = ops.token_scores_workspace(300, 50_000, 20)
    if need:
        x = logits(300, 50_000, torch.bfloat16, seed=1)
        with pytest.raises(ValueError):
            ops.token_scores(x, None, 20, workspace=torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
