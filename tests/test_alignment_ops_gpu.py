"""GPU: scoring, preference and policy losses, the scaled embedding and the 8-bit linear layer against plain statements in 64 bits.

Tolerances.  H = 2^-24 is half a step of f32, finfo(t).eps / 2 of a result's type t.  A row's sum of exponentials carries the rounding of its
terms' arguments (x - m and, for bf16 rows, times log2 e: |x - m| H each, weighted by the softmax: <= ~11 on average for 110,000 logits), of
the exponentials (2 H) and of the adding-up (a thread's chain of <= 13 chunks of 8, 6 + 4 tree steps: <= 130 H if all went one way, a few H
in fact): 160 H covers them; the label's own x_y - m and the logarithm add 2 |logp| H.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
H = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16]


def half_step(dt):
    return torch.finfo(dt).eps / 2


def make_rows(N, T, V, dt, pitch=None, seed=0, masked=True, ninf=False, offset=0):
    """Logits [N, T, V] in a buffer of NaN (pitch > V: NaN columns behind), labels with uncounted positions whose rows are NaN."""
    g = torch.Generator().manual_seed(1000 * V + 10 * N + T + seed)
    pitch = pitch or V
    x = (torch.randn(N, T, V, generator=g) * 3).to(dt)
    labels = torch.randint(0, V, (N, T), generator=g)
    x.scatter_add_(2, labels[..., None], torch.full((N, T, 1), 4.0, dtype=dt))
    if ninf and V > 2:
        x[:, :, V // 2] = float("-inf")
        labels[labels == V // 2] = V - 1
    if masked:
        flat = labels.view(-1)
        for i, bad in zip(range(0, flat.numel(), 5), [-100, V, -1, 2 ** 40, -2 ** 40] * (flat.numel() // 5 + 1)):
            flat[i] = bad
        if N > 2:
            labels[1] = -100
    keep = (labels >= 0) & (labels < V)
    x[~keep] = float("nan")
    buf = torch.full((N * T * pitch + offset + 64,), float("nan"), dtype=dt)
    view = buf[offset:offset + N * T * pitch].view(N, T, pitch)[:, :, :V]
    view.copy_(x)
    buf = buf.cuda()
    return buf[offset:offset + N * T * pitch].view(N, T, pitch)[:, :, :V], labels.cuda(), buf


def plain(x, labels):
    """64 bits: keep, label index, logp (0 where not counted), softmax"""
    x = x.double()
    V = x.shape[-1]
    keep = (labels >= 0) & (labels < V)
    x = torch.where(keep[..., None], x, torch.zeros_like(x))
    lab = torch.where(keep, labels, torch.zeros_like(labels))
    lp = torch.log_softmax(x, -1)
    own = lp.gather(-1, lab[..., None])[..., 0] * keep
    return keep, lab, own, lp.exp()


def lp_tol(own):
    return H * (2 * own.abs() + 160)


def dl_expect(p, lab, keep, coef):
    d = -p * coef[..., None]
    d.scatter_add_(-1, lab[..., None], coef[..., None])
    return torch.where(keep[..., None], d, torch.zeros_like(d))


def check_dl(got, p, lab, keep, coef, mag, dt, logp):
    """got against coef (onehot - p): every factor of the product carries the row's relative error, the coefficient that of its parts (mag)."""
    want = dl_expect(p, lab, keep, coef)
    rel = H * (4 * logp.abs() + 400)[..., None]
    one = torch.zeros_like(p).scatter_(-1, lab[..., None], 1.0)
    tol = mag[..., None] * rel * (p + one) + want.abs() * half_step(dt) + torch.finfo(dt).tiny
    bad = ((got.double() - want).abs() > tol) & keep[..., None]
    assert not bad.any(), ((got.double() - want).abs() / tol)[bad].max().item()
    assert (got[~keep] == 0).all()


SIZES = [(1, 1, 1), (2, 3, 2), (3, 5, 64), (2, 9, 1009), (2, 4, 2049), (3, 3, 9001), (2, 3, 30011), (2, 3, 50265), (1, 3, 60001), (1, 2, 110003)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("size", SIZES)
def test_token_logprob_and_gradient(size, dt):
    from multimodalsum_amd import kernels as kn
    N, T, V = size
    for pitch, offset, ninf in ((V, 0, False), ((V + 127) // 128 * 128, 0, True), (V + 3, 1, True)):
        x, labels, _ = make_rows(N, T, V, dt, pitch, ninf=ninf, offset=offset, masked=N * T > 2)
        keep, lab, own, p = plain(x, labels)
        stats = torch.full((N, T, 2), float("nan"), device="cuda")
        logp = kn.token_logprob(x, labels, stats)
        assert ((logp.double() - own).abs() <= lp_tol(own)).all()
        assert (logp[~keep] == 0).all()
        assert torch.equal(logp, kn.token_logprob(x, labels))
        for coef in (torch.linspace(-1.5, 2.0, N * T, device="cuda").view(N, T), torch.linspace(0.5, -1.0, N, device="cuda")):
            alpha = torch.tensor([0.75], device="cuda")
            got = kn.token_logprob_bwd(x, labels, stats, coef, alpha)
            c = 0.75 * (coef if coef.dim() == 2 else coef[:, None].expand(N, T)).double()
            check_dl(got, p, lab, keep, c, c.abs(), dt, own)


def test_extreme_logits():
    """-inf everywhere but the label: probability one, no gradient; the label itself at -inf: -inf with a finite gradient; huge logits; a NaN gives NaN."""
    from multimodalsum_amd import kernels as kn
    for dt in DTYPES:
        for V in (8, 1009, 50265, 110003):
            x = torch.randn(1, 5, V, device="cuda").to(dt)
            x[0, 0] = float("-inf")
            x[0, 0, 3] = 1.5
            x[0, 1, 3] = float("-inf")
            x[0, 2] *= 1e4
            x[0, 3, V - 1] = float("nan")
            x[0, 4] = float("-inf")
            labels = torch.full((1, 5), 3, device="cuda")
            stats = torch.empty(1, 5, 2, device="cuda")
            lp = kn.token_logprob(x, labels, stats)[0]
            want = torch.log_softmax(x[0].double(), -1)[:, 3]
            assert lp[0] == 0 and lp[1] == float("-inf") and torch.isnan(lp[3]) and torch.isnan(lp[4])
            assert (lp[2] - want[2]).abs() <= lp_tol(want[2])
            d = kn.token_logprob_bwd(x, labels, stats, torch.ones(1, 5, device="cuda"))[0].double()
            assert (d[0] == 0).all() and torch.isfinite(d[1]).all() and (d[1].sum()).abs() < 0.02 and d[1, 3] == 1
            assert torch.isfinite(d[2]).all()


def pref_plain(own, keep, ref, beta, eps, average):
    P = own.shape[0] // 2
    cnt = keep.sum(1).clamp(min=1).double()
    leaf = own.clone().requires_grad_(True)
    S = leaf.sum(1) / (cnt if average else 1.0)
    r = S - (ref.double() if ref is not None else 0.0)
    h = beta * (r[:P] - r[P:])
    F = torch.nn.functional
    loss = -((1 - eps) * F.logsigmoid(h) + eps * F.logsigmoid(-h)).mean()
    loss.backward()
    return loss.detach(), h.detach(), S.detach(), leaf.grad * keep


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("eps", [0.0, 0.1])
@pytest.mark.parametrize("size", [(2, 1, 5), (4, 7, 1009), (6, 33, 2050), (4, 5, 50265), (2, 1100, 5), (66, 1000, 3)])
def test_preference_loss(size, eps, average, dt):
    import multimodalsum_amd as mm
    from multimodalsum_amd import kernels as kn
    N, T, V = size
    beta = 0.1
    for with_ref in (True, False):
        x, labels, buf = make_rows(N, T, V, dt, V + 7, masked=T > 1)
        keep, lab, own, p = plain(x, labels)
        ref = (-0.7 * T * torch.rand(N, device="cuda") / (T if average else 1)) if with_ref else None
        loss, h, S, coef = pref_plain(own, keep, ref, beta, eps, average)
        # S: T terms; h: beta times the difference of two S and two refs; loss: 1-Lipschitz in h; coef = beta / P (eps - sigmoid(-h)) / cnt
        s_tol = (lp_tol(own) * keep).sum(1) + H * T * own.abs().sum(1)
        h_tol = beta * (2 * s_tol.max() + 4 * H * (S.abs().max() + (0 if ref is None else ref.abs().max().double()))) + 4 * H * h.abs().max()
        mag = torch.full_like(own, 0.0) + coef.abs() + (h_tol / (H * 400)) * beta / (N // 2)
        got = kn.preference_loss(x, labels, ref, beta, eps, average)
        assert ((got[2].double() - S).abs() <= s_tol + 2 * H * S.abs()).all()
        assert ((got[1].double() - h).abs() <= h_tol).all()
        assert (got[0].double() - loss).abs() <= h_tol + 16 * H * (1 + loss.abs())
        check_dl(got[3], p, lab, keep, coef, mag, dt, own)
        # the module: the same numbers, the upstream gradient applied
        xg = x.clone().requires_grad_(True)
        m = mm.PreferenceLoss(beta, eps, average)
        l2 = m(xg, labels, ref)
        assert torch.equal(l2.detach(), got[0]) and torch.equal(m.margins, got[1])
        (l2 * 0.5).backward()
        check_dl(xg.grad, p, lab, keep, 0.5 * coef, mag, dt, own)
        # over the logits themselves, and beside them with padding columns
        wide = torch.full((N, T, V + 5), float("nan"), dtype=dt, device="cuda")
        _, _, d = mm.preference_loss_and_grad(x, labels, ref, beta=beta, label_smoothing=eps, average=average, dlogits=wide)
        assert torch.equal(d[:, :, :V], got[3]) and (d[:, :, V:] == 0).all()
        tail = buf[N * T * (V + 7):].clone()
        pad = buf[:N * T * (V + 7)].view(N, T, V + 7)[:, :, V:].clone()
        _, _, d = mm.preference_loss_and_grad(x, labels, ref, beta=beta, label_smoothing=eps, average=average, dlogits=x)
        assert d.data_ptr() == x.data_ptr() and torch.equal(d, got[3])
        assert torch.isnan(buf[N * T * (V + 7):]).all() and torch.isnan(tail).all() and torch.isnan(buf[:N * T * (V + 7)].view(N, T, V + 7)[:, :, V:]).all() and torch.isnan(pad).all()


def policy_plain(own, keep, old, adv, ref, lo, hi, kl_coef, reduction):
    N, T = own.shape
    leaf = own.clone().requires_grad_(True)
    a = (adv if adv.dim() == 2 else adv[:, None].expand(N, T)).double()
    ratio = torch.where(keep, (leaf - torch.nan_to_num(old.double())).exp(), torch.ones_like(leaf))
    w = keep / (keep.sum().clamp(min=1) if reduction == "token" else keep.sum(1, keepdim=True).clamp(min=1) * N).double()
    l1, l2 = -a * ratio, -a * ratio.clamp(1 - lo, 1 + hi)
    kl = torch.zeros_like(own)
    if ref is not None:
        d = torch.where(keep, torch.nan_to_num(ref.double()) - leaf, torch.zeros_like(leaf))
        kl = d.exp() - d - 1
    loss = (w * (torch.maximum(l1, l2) + kl_coef * kl)).sum()
    loss.backward()
    mag = w * (a.abs() * ratio.detach() + kl_coef * (1 + (kl.detach() + 1).abs() * 2))
    return loss.detach(), (w * kl).sum().detach(), (w * (l1 < l2)).sum().detach(), leaf.grad * keep, mag


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("kl_coef", [0.0, 0.1])
@pytest.mark.parametrize("size", [(1, 1, 5), (5, 7, 1009), (3, 70, 300), (3, 4, 50265), (2, 2, 110003), (2, 2100, 7)])
def test_policy_loss(size, kl_coef, reduction, dt):
    import multimodalsum_amd as mm
    N, T, V = size
    for per_token in (False, True):
        x, labels, buf = make_rows(N, T, V, dt, V + 7, masked=N * T > 1, offset=1)
        keep, lab, own, p = plain(x, labels)
        g = torch.Generator().manual_seed(V)
        step = (torch.randn(N, T, generator=g) * 0.3).cuda()
        for edge in (0.8, 1.28):                                   # the bounded branch switches there: stay a rounding away
            step[(step.exp() - edge).abs() < 1e-3] = 0.0
        old = torch.where(keep, own.float() - step, torch.full_like(step, float("nan")))
        ref = torch.where(keep, own.float() + 0.4 * step.flip(0), torch.full_like(step, float("nan"))) if kl_coef else None
        adv = torch.randn((N, T) if per_token else (N,), generator=g).cuda()
        if N > 2:
            adv.view(-1)[0] = 0.0
        loss, kl, clipped, coef, mag = policy_plain(own, keep, old, adv, ref, 0.2, 0.28, kl_coef, reduction)
        l, k, c, tok, d = mm.policy_loss_and_grad(x, labels, old, adv, ref, clip_low=0.2, clip_high=0.28, kl_coef=kl_coef, reduction=reduction)
        # a token's terms carry |error of logp| (times the magnitudes of its parts) and a few roundings; the mean adds N T of them
        t_tol = (mag * (lp_tol(own) + H * (4 * own.abs() + 16))).sum() + 32 * H * mag.sum()
        assert ((tok.double() - own).abs() <= lp_tol(own)).all()
        assert (l.double() - loss).abs() <= t_tol + 8 * H * loss.abs() and (c.double() - clipped).abs() <= 32 * H
        assert (k.double() - kl).abs() <= (t_tol / max(kl_coef, 1e-9) if kl_coef else 0.0) + 8 * H
        check_dl(d, p, lab, keep, coef, mag, dt, own)
        xg = x.clone().requires_grad_(True)
        m = mm.ClippedPolicyLoss(0.2, 0.28, kl_coef, reduction)
        l2 = m(xg, labels, old, adv, ref)
        assert (l2 - l).abs() <= 2 * t_tol + 8 * H * loss.abs() and torch.equal(m.logps, tok)
        (l2 * 3.0).backward()
        check_dl(xg.grad, p, lab, keep, 3 * coef, 3 * mag, dt, own)
        l3, _, _, tok3, d3 = mm.policy_loss_and_grad(x, labels, old, adv, ref, clip_low=0.2, clip_high=0.28, kl_coef=kl_coef, reduction=reduction, dlogits=x)
        assert torch.equal(l3, l) and torch.equal(tok3, tok) and torch.equal(d3, d) and d3.data_ptr() == x.data_ptr()
        assert torch.isnan(buf[1 + N * T * (V + 7):]).all() and torch.isnan(buf[1:1 + N * T * (V + 7)].view(N, T, V + 7)[:, :, V:]).all() and torch.isnan(buf[0])


def test_losses_with_nothing_counted():
    import multimodalsum_amd as mm
    for dt in DTYPES:
        x = torch.full((4, 3, 1009), float("nan"), dtype=dt, device="cuda")
        labels = torch.full((4, 3), -100, device="cuda")
        z = torch.full((4, 3), float("nan"), device="cuda")
        l, kl, c, tok, d = mm.policy_loss_and_grad(x, labels, z, torch.ones(4, device="cuda"), z, kl_coef=0.1)
        assert l == 0 and kl == 0 and c == 0 and (tok == 0).all() and (d == 0).all()
        l, h, d = mm.preference_loss_and_grad(x, labels, None)
        assert (l - math.log(2.0)).abs() < 4 * H and (h == 0).all() and (d == 0).all()
        seq, tok = mm.sequence_logprobs(x, labels, average=True)
        assert (seq == 0).all() and (tok == 0).all()


def test_gradient_against_differences():
    """The losses' directional derivatives in f32 against central differences of the 64-bit statement on the same logits."""
    import multimodalsum_amd as mm
    x, labels, _ = make_rows(4, 6, 257, torch.float32, masked=True)
    x = torch.nan_to_num(x.contiguous())
    g = torch.Generator().manual_seed(5)
    v = torch.randn(4, 6, 257, generator=g).cuda().double()
    ref = torch.randn(4, generator=g).cuda()
    keep, _, own, _ = plain(x, labels)
    old, adv, rtok = (own + 0.05).float(), torch.randn(4, generator=g).cuda(), (own - 0.2).float()

    def pref(z):
        k, _, o, _ = plain(z, labels)
        return pref_plain(o, k, ref, 0.3, 0.1, True)[0]

    def pol(z):
        k, _, o, _ = plain(z, labels)
        return policy_plain(o, k, old, adv, rtok, 0.2, 0.2, 0.3, "token")[0]

    _, _, d1 = mm.preference_loss_and_grad(x, labels, ref, beta=0.3, label_smoothing=0.1, average=True)
    d2 = mm.policy_loss_and_grad(x, labels, old, adv, rtok, kl_coef=0.3)[4]
    e = 1e-4
    for f, d in ((pref, d1), (pol, d2)):
        diff = (f(x.double() + e * v) - f(x.double() - e * v)) / (2 * e)
        # f32 gradient: 2^-24 scale per element against |v| ~ 1; differences: e^2 third derivatives and 64-bit cancellation 1e-16 / e
        assert (diff - (d.double() * v).sum()).abs() <= 400 * H * (d.double() * v).abs().sum() + 1e-6


# ---------------------------------------------------------------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------------------------------------------------------------
EMB = [(1, 1, 1), (7, 5, 3), (21, 1009, 256), (1000, 50, 100), (4097, 70000, 64), (5000, 300, 777), (300, 50265, 1024), (12000, 1, 40), (9000, 255, 512), (4096, 256, 8),
       (40000, 2, 520), (2500, 4000, 16), (300000, 1000, 8)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("case", EMB)
def test_embedding(case, dt):
    import multimodalsum_amd as mm
    n, V, D = case
    g = torch.Generator().manual_seed(n + V + D)
    ids = (torch.rand(n, generator=g) ** 3 * V).long()              # skewed: frequent ids cross many stretches
    if n > 20:
        ids[3], ids[5], ids[7], ids[9] = -1, V, 2 ** 40, -2 ** 40
        ids[n // 3:n // 2] = V - 1
    ids = ids.cuda()
    table = torch.randn(V, D, generator=g).to(dt).cuda()
    dy = torch.randn(n, D, generator=g).to(dt).cuda()
    scale, pad = 5.5, (0 if V > 1 else None)
    ok = (ids >= 0) & (ids < V)
    y = mm.scaled_embedding(ids, table, scale)
    want = torch.where(ok[:, None], table.double()[torch.where(ok, ids, torch.zeros_like(ids))] * scale, 0.0)
    assert ((y.double() - want).abs() <= want.abs() * half_step(dt) + H * want.abs()).all()
    live = ok & (ids != pad) if pad is not None else ok
    il, dl = ids[live].cpu(), dy[live].double().cpu()
    want = torch.zeros(V, D, dtype=torch.float64).index_add_(0, il, dl).cuda() * scale
    mass = torch.zeros(V, D, dtype=torch.float64).index_add_(0, il, dl.abs()).cuda() * scale
    # chains of at most 32 inside a stretch, then a quarter of the stretches in a row, 2 + 1 more: each adds H of the partial sums
    tol = mass * H * (32 + n / 128 + 8)
    d = mm.scaled_embedding_grad(dy, ids, V, scale, padding_idx=pad)
    assert d.dtype == torch.float32 and ((d.double() - want).abs() <= tol).all()
    assert (d[mass.sum(1) == 0] == 0).all()
    assert torch.equal(d, mm.scaled_embedding_grad(dy, ids, V, scale, padding_idx=pad))
    base = torch.randn(V, D, generator=g).cuda()
    acc = base.clone()
    assert mm.scaled_embedding_grad(dy, ids, V, scale, padding_idx=pad, out=acc, accumulate=True).data_ptr() == acc.data_ptr()
    untouched = mass.sum(1) == 0
    assert torch.equal(acc[untouched], base[untouched]) and ((acc.double() - base.double() - want).abs() <= tol + 2 * H * (base.abs().double() + mass)).all()
    # strided dy and table rows; rows that start anywhere
    wide = torch.full((n, D + 3), float("nan"), dtype=dt, device="cuda")
    wide[:, 1:D + 1] = dy
    assert ((mm.scaled_embedding_grad(wide[:, 1:D + 1], ids, V, scale, padding_idx=pad).double() - want).abs() <= tol).all()
    tw = torch.full((V, D + 3), float("nan"), dtype=dt, device="cuda")
    tw[:, 1:D + 1] = table
    assert torch.equal(mm.scaled_embedding(ids, tw[:, 1:D + 1], scale), y)
    # autograd
    t = table.clone().requires_grad_(True)
    mm.scaled_embedding(ids.view(1, n), t, scale, pad).backward(dy.view(1, n, D))
    assert torch.equal(t.grad, d.to(dt))


def test_repeated_rows():
    """A gradient that is one row for every position (sum over positions) and activations that are one row for every token: strides of zero."""
    import multimodalsum_amd as mm
    table = torch.randn(50, 24, device="cuda", requires_grad=True)
    ids = torch.arange(100, device="cuda") % 50
    v = torch.randn(24, device="cuda")
    (mm.scaled_embedding(ids, table, 3.0).sum(0) * v).sum().backward()
    assert torch.equal(table.grad, (v * 2 * 3.0).expand(50, 24))
    lin = mm.Int8Linear(torch.randn(20, 24, device="cuda"))
    assert torch.equal(lin(v.expand(7, 24)), lin(v).expand(7, 20))


def test_embedding_without_ids_and_module():
    import multimodalsum_amd as mm
    ids = torch.empty(0, 3, dtype=torch.int64, device="cuda")
    table = torch.randn(11, 8, device="cuda")
    assert mm.scaled_embedding(ids, table, 2.0).shape == (0, 3, 8)
    out = torch.full((11, 8), 7.0, device="cuda")
    dy = torch.empty(0, 3, 8, device="cuda")
    assert (mm.scaled_embedding_grad(dy, ids, 11, out=out, accumulate=True) == 7).all()
    assert (mm.scaled_embedding_grad(dy, ids, 11, out=out) == 0).all()
    m = mm.ScaledEmbedding(11, 8, scale=4.0, padding_idx=1)
    y = m(torch.tensor([[1, 2, 2]], device="cuda"))
    assert (y[0, 0] == 0).all() and torch.equal(y[0, 1], 4.0 * m.weight[2])
    y.sum().backward()
    assert (m.weight.grad[2] == 8).all() and (m.weight.grad[[0, 1, 3]] == 0).all()


# ---------------------------------------------------------------------------------------------------------------------------------
# 8-bit linear layer
# ---------------------------------------------------------------------------------------------------------------------------------
def quantize_plain(x):
    x = x.double()
    top = x.abs().amax(1)
    q = torch.where(top[:, None] > 0, torch.round((x * 127.0) / top[:, None]), torch.zeros_like(x))
    return q, (top / 127.0).float()                                  # 64-bit quotient, rounded once (a 32-bit division by a scalar multiplies by its reciprocal)


def linear_plain(x, w, bias, gelu):
    qx, sx = quantize_plain(x)
    qw, sw = quantize_plain(w)
    y = torch.mm(qx, qw.t().contiguous()) * sx.double()[:, None] * sw.double()
    mag = y.abs()
    if bias is not None:
        y = y + bias.double()
        mag = mag + bias.double().abs()
    if gelu:
        y = 0.5 * y * (1 + torch.erf(y / math.sqrt(2.0)))
    return y, mag


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 17), (5, 128), (70, 1000), (9, 4096), (2, 20011)])
def test_quantize_rows(M, K, dt):
    from multimodalsum_amd import kernels as kn
    g = torch.Generator().manual_seed(K)
    x = torch.randn(M, K, generator=g) * torch.logspace(-30, 30, M).unsqueeze(1)
    x[0, : K // 2] = 0.5 * x[0].abs().max()                         # 63.5: a tie, to even
    if M > 2:
        x[1] = 0.0
        x[2, 0] = torch.finfo(torch.float32).max if dt == torch.float32 else 3e38
    x = x.to(dt).cuda()
    q, s = kn.quantize_rows(x)
    want, ws = quantize_plain(x)
    assert q.shape[1] % kn.I8_K_STEP == 0 and (q[:, K:] == 0).all() and torch.equal(s, ws)
    diff = (q[:, :K].double() - want).abs()
    if dt == torch.bfloat16:
        assert diff.max() == 0                                       # 15-bit products by 8-bit maxima: no quotient is that near a tie without being one
    else:
        off = diff > 0                                               # the f32 quotient (two roundings) may round onto a tie that the exact one misses
        frac = ((x.double() * 127.0 / x.double().abs().amax(1, keepdim=True)) - 0.5) % 1.0
        assert diff.max() <= 1 and (torch.minimum(frac, 1 - frac)[off] <= 128 * 2 * H).all()
    pad = torch.full((M, K + 5), float("nan"), dtype=dt, device="cuda")
    pad[:, 3:K + 3] = x
    q2, s2 = kn.quantize_rows(pad[:, 3:K + 3])
    assert torch.equal(q, q2) and torch.equal(s, s2)


I8 = [(1, 17, 16), (1, 1, 1), (3, 64, 100), (8, 1024, 1024), (16, 50, 4096), (17, 129, 257), (32, 5001, 1024), (33, 1024, 2000), (65, 200, 64), (128, 512, 512), (129, 1000, 640),
      (257, 255, 384), (1152, 1024, 1024), (1300, 2051, 128), (700, 4096, 1024),
      (4100, 2100, 384), (33000, 70, 128), (300, 33001, 256), (2048, 4096, 1024), (8200, 1028, 128), (2500, 4100, 1024), (40000, 256, 512)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M,N,K", I8)
def test_int8_linear(M, N, K, dt):
    from multimodalsum_amd import Int8Linear
    g = torch.Generator().manual_seed(M + N + K)
    x = (torch.randn(M, K, generator=g) * (0.2 + torch.rand(M, 1, generator=g))).to(torch.bfloat16).to(dt).cuda()      # bf16 values: quotients off the ties
    w = (torch.randn(N, K, generator=g) * 0.05).to(torch.bfloat16).cuda()
    bias = torch.randn(N, generator=g).cuda()
    for b, gelu in ((None, False), (bias, False), (bias, True)):
        want, mag = linear_plain(x, w, b, gelu)
        for out in DTYPES:
            y = Int8Linear(w, b, gelu=gelu, out_dtype=out)(x)
            assert y.dtype == out and y.shape == (M, N)
            # int -> f32, two scales, the bias: 4 H of the parts; GELU (slope <= 1.13): the same and the error function's 2^-22 |y|
            tol = mag * (8 if not gelu else 40) * H + want.abs() * half_step(out) + torch.finfo(out).tiny
            assert ((y.double() - want).abs() <= tol).all(), ((y.double() - want).abs() / tol).max().item()


@pytest.mark.parametrize("M,N,K", [(2305, 2100, 384), (2500, 6500, 900), (129, 60000, 300), (573, 12001, 700), (4353, 4099, 2600), (3100, 4100, 1000), (8100, 2040, 60), (4099, 7000, 300),
                                   (8000, 8001, 1100)])
@pytest.mark.parametrize("out", DTYPES)
def test_int8_product_at_tile_edges(M, N, K, out):
    """The large tiles, several to a workgroup too, with rows, columns and k behind the last whole tile; nothing is written around the result."""
    from multimodalsum_amd import kernels as kn
    g = torch.Generator(device="cuda").manual_seed(M + K)
    Kp = -(-K // kn.I8_K_STEP) * kn.I8_K_STEP
    qx = torch.zeros(M, Kp, dtype=torch.int8, device="cuda")
    qw = torch.zeros(N, Kp, dtype=torch.int8, device="cuda")
    qx[:, :K] = torch.randint(-127, 128, (M, K), generator=g, device="cuda")
    qw[:, :K] = torch.randint(-127, 128, (N, K), generator=g, device="cuda")
    sx, sw, bias = (torch.rand(n, generator=g, device="cuda") for n in (M, N, N))
    want = torch.mm(qx.double(), qw.double().t().contiguous()) * sx.double()[:, None] * sw.double()
    for b, gelu in ((None, False), (bias, False), (bias, True)):
        ref = want if b is None else want + b.double()
        tol = (want.abs() + 1) * (8 if not gelu else 40) * H         # as for the linear layer; the bias is below 1
        if gelu:
            ref = 0.5 * ref * (1 + torch.erf(ref / math.sqrt(2.0)))
        wide = torch.full((M + 2, N + 6), float("nan"), dtype=out, device="cuda")
        kn.gemm_i8(qx, sx, qw, sw, wide[1:-1, 3:N + 3], b, gelu)
        y = wide[1:-1, 3:N + 3].double()
        assert ((y - ref).abs() <= tol + ref.abs() * half_step(out) + torch.finfo(out).tiny).all()
        assert torch.isnan(wide[0]).all() and torch.isnan(wide[-1]).all() and torch.isnan(wide[:, :3]).all() and torch.isnan(wide[:, N + 3:]).all()


def test_int8_linear_extremes_and_shapes():
    from multimodalsum_amd import Int8Linear
    g = torch.Generator().manual_seed(3)
    w = torch.randn(48, 96, generator=g).cuda()
    w[5] = 0.0
    bias = torch.randn(48, generator=g).cuda()
    lin = Int8Linear(w, bias)
    x = torch.randn(2, 3, 96, generator=g).cuda()
    x[0, 0] = 0.0
    x[0, 1, 4] = float("inf")
    x[0, 2, 9] = float("nan")
    y = lin(x)
    assert y.shape == (2, 3, 48) and torch.equal(y[0, 0], bias) and torch.isnan(y[0, 1:]).all() and torch.isfinite(y[1]).all()
    assert torch.equal(y[1][:, 5], bias[5].expand(3))
    assert lin(x[:, :, :][:0]).shape == (0, 3, 48) and torch.equal(lin(x[1, 2]), y[1, 2])
    assert torch.equal(lin(x.transpose(0, 1))[:, 1], y[1])          # rows that are not packed
    # the largest sums: all values at 127
    big = Int8Linear(torch.ones(33, 131072, device="cuda"))
    assert torch.equal(big(torch.ones(2, 131072, device="cuda")), ((torch.tensor(1.0) / 127) ** 2 * float(127 * 127 * 131072)).cuda().expand(2, 33).contiguous()) or \
        (big(torch.ones(2, 131072, device="cuda")) - 131072.0).abs().max() <= 131072 * 6 * H
    emb = Int8Linear.from_linear(torch.nn.Linear(96, 48, device="cuda"))
    assert emb.state_dict().keys() == {"qweight", "scale", "bias"}
    # operands that are views of wider ones, for each of the products
    from multimodalsum_amd import kernels as kn
    for M, N in ((5, 40), (100, 200), (2500, 4100)):
        a, b = torch.randint(-127, 128, (M, 384), dtype=torch.int8, generator=g).cuda(), torch.randint(-127, 128, (N, 512), dtype=torch.int8, generator=g).cuda()
        one = torch.ones(max(M, N), device="cuda")
        got = kn.gemm_i8(a[:, 128:], one[:M], b[:, 128:384], one[:N], torch.empty(M, N, device="cuda"))
        assert torch.equal(got.double(), torch.mm(a[:, 128:].double(), b[:, 128:384].double().t().contiguous()))      # sums below 2^24
    # columns and rows behind the result stay as they were
    q, s = kn.quantize_rows(x[1])
    out = torch.full((8, 60), float("nan"), device="cuda")
    kn.gemm_i8(q, s, lin.qweight, lin.scale, out[2:5, 4:52], lin.bias)
    assert torch.equal(out[2:5, 4:52], y[1]) and torch.isnan(out[:2]).all() and torch.isnan(out[5:]).all() and torch.isnan(out[:, :4]).all() and torch.isnan(out[:, 52:]).all()


# ---------------------------------------------------------------------------------------------------------------------------------
# together; streams; graphs
# ---------------------------------------------------------------------------------------------------------------------------------
def test_preference_step_with_a_frozen_8bit_model():
    """A tied embedding / vocabulary model: look up, score the pair under the frozen 8-bit copy, preference loss, gradients back to the table by both ways."""
    import multimodalsum_amd as mm
    g = torch.Generator().manual_seed(11)
    V, D, N, T = 1009, 64, 6, 9
    emb = mm.ScaledEmbedding(V, D, scale=8.0, padding_idx=1)
    with torch.no_grad():
        emb.weight.copy_((torch.randn(V, D, generator=g) * 0.1).cuda())
        emb.weight[1].zero_()
    ids = torch.randint(2, V, (N, T), generator=g).cuda()
    ids[1, 5:] = 1
    labels = torch.where(ids == 1, torch.full_like(ids, -100), ids).roll(-1, 1)
    labels[:, -1] = -100
    head = mm.Int8Linear(emb.weight)
    with torch.no_grad():
        ref, _ = mm.sequence_logprobs(head(mm.scaled_embedding(ids, emb.weight, 8.0)), labels)
    hidden = emb(ids)
    logits = torch.matmul(hidden.reshape(-1, D), emb.weight.t()).view(N, T, V)
    loss = mm.PreferenceLoss(beta=0.2)(logits, labels, ref)
    loss.backward()
    # 64 bits, with the 8-bit model's scores as given
    w = emb.weight.detach().double().requires_grad_(True)
    h = w[ids] * 8.0
    h = torch.where((ids == 1)[..., None], h.detach(), h)
    x = h @ w.t()
    keep = labels >= 0
    lp = torch.log_softmax(x, -1).gather(-1, labels.clamp(min=0)[..., None])[..., 0] * keep
    S = lp.sum(1)
    hh = 0.2 * ((S[:3] - ref[:3].double()) - (S[3:] - ref[3:].double()))
    want = -torch.nn.functional.logsigmoid(hh).mean()
    want.backward()
    assert (loss.double() - want).abs() < 1e-4 and (emb.weight.grad.double() - w.grad).abs().max() < 1e-4 * w.grad.abs().max()
    exact = torch.log_softmax((h @ w.t()).detach(), -1).gather(-1, labels.clamp(min=0)[..., None])[..., 0] * keep
    assert (ref.double() - exact.sum(1)).abs().max() < 0.05 * exact.sum(1).abs().max()      # 8 bits: a few per cent of a score


def test_tuning_the_summariser():
    """The framework's decoder under both losses: the parameters' gradients equal those of the same losses written in torch on the same logits."""
    import multimodalsum_amd as mm
    from multimodalsum_amd.modules import BartForEncConditionalGeneration, init_formula
    from multimodalsum_amd.selftest import tiny_config
    cfg = tiny_config()

    def fresh():
        m = BartForEncConditionalGeneration(cfg, device="cuda:0", dtype=torch.float32, deterministic=True)
        init_formula(m)
        m._engine.mark_weights_changed()
        return m.train()

    g = torch.Generator().manual_seed(2)
    hid = (torch.randn(4, 2, 6, cfg.d_model, generator=g) * 0.5).cuda()
    labels = torch.randint(4, cfg.vocab_size, (4, 9), generator=g).cuda()
    labels[1, 6:] = cfg.pad_token_id
    counted = torch.where(labels == cfg.pad_token_id, torch.full_like(labels, -100), labels)
    rd = torch.zeros(4, 1, device="cuda")
    with torch.no_grad():
        first = fresh()(hid, rd, labels=labels)[0]
        ref, old = mm.sequence_logprobs(first, counted)
    ref, old, rtok, adv = ref - torch.arange(4.0, device="cuda"), old - 0.1, old + 0.2, torch.tensor([1.0, -0.5, 0.3, -2.0], device="cuda")

    def in_torch(kind, logits):
        keep = counted >= 0
        lp = torch.log_softmax(logits.double(), -1).gather(-1, counted.clamp(min=0)[..., None])[..., 0] * keep
        if kind == "pref":
            r = lp.sum(1) - ref.double()
            return -torch.nn.functional.logsigmoid(0.5 * (r[:2] - r[2:])).mean()
        ratio, d = (lp - old.double()).exp(), (rtok.double() - lp)
        a = adv.double()[:, None]
        t = torch.maximum(-a * ratio, -a * ratio.clamp(0.8, 1.2)) + 0.1 * (d.exp() - d - 1)
        return (t * keep).sum() / keep.sum()

    pref, pol = mm.PreferenceLoss(beta=0.5), mm.ClippedPolicyLoss(kl_coef=0.1)
    for kind, loss in (("pref", lambda x: pref(x, counted, ref)), ("pol", lambda x: pol(x, counted, old, adv, rtok))):
        results = []
        for f in (loss, lambda x: in_torch(kind, x)):
            model = fresh()
            value = f(model(hid, rd, labels=labels)[0])
            value.backward()
            results.append((value.detach().double(), {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}))
        (v1, g1), (v2, g2) = results
        assert (v1 - v2).abs() < 1e-5 * (1 + v2.abs()) and g1.keys() == g2.keys() and len(g1) > 10
        for n in g1:                                                # f32 gradients of one model from logits' gradients that agree to f32
            assert (g1[n] - g2[n]).abs().max() <= 1e-4 * g2[n].abs().max() + 1e-7, n


def all_ops(s):
    import multimodalsum_amd as mm
    seq, tok = mm.sequence_logprobs(s["x"], s["labels"])
    p = mm.preference_loss_and_grad(s["x"], s["labels"], s["ref"])
    q = mm.policy_loss_and_grad(s["x"], s["labels"], s["old"], s["adv"], s["old"], kl_coef=0.1)
    y = mm.scaled_embedding(s["ids"], s["table"], 2.0)
    d = mm.scaled_embedding_grad(s["dy"], s["ids"], s["table"].shape[0], 2.0)
    return [seq, tok, *p, *q, y, d, s["lin"](s["act"]), s["lin"](s["act"][:5]), s["lin2"](s["act2"])]


def op_state(seed, n=5000):
    import multimodalsum_amd as mm
    x, labels, _ = make_rows(4, 8, 1009, torch.bfloat16, seed=seed)
    g = torch.Generator().manual_seed(seed)
    return dict(x=torch.nan_to_num(x), labels=labels, ref=torch.randn(4, generator=g).cuda(), old=torch.randn(4, 8, generator=g).cuda() - 3, adv=torch.randn(4, generator=g).cuda(),
                ids=torch.randint(0, 700, (n,), generator=g).cuda(), table=torch.randn(700, 64, generator=g).cuda(), dy=torch.randn(n, 64, generator=g).cuda(),
                lin=mm.Int8Linear(torch.randn(300, 256, generator=g).cuda()), act=torch.randn(150, 256, generator=g).cuda(),
                lin2=mm.Int8Linear(torch.randn(1024, 384, generator=g).cuda()), act2=torch.randn(9216, 384, generator=g).cuda())


def test_graph_replay():
    """Captured once, replayed on new inputs between eager calls; two graphs replayed in turn share nothing."""
    for n in (300, 5000):
        states = [op_state(1, n), op_state(2, n)]
        graphs = []
        for s in states:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                all_ops(s)
            torch.cuda.current_stream().wait_stream(side)
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                out = all_ops(s)
            graphs.append((gr, out))
        for rep in range(3):
            for s in states:
                s["x"].mul_(1.1)
                s["dy"].add_(0.25)
                s["act"].mul_(-0.9)
            want = [[t.clone() for t in all_ops(s)] for s in states]
            for gr, _ in graphs:
                gr.replay()
            torch.cuda.synchronize()
            for (gr, out), w in zip(graphs, want):
                for a, b in zip(out, w):
                    assert torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float()))


def test_two_streams():
    states = [op_state(3), op_state(4)]
    want = [[t.clone() for t in all_ops(s)] for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for s, st in zip(states, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(all_ops(s))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(torch.nan_to_num(x.float()), torch.nan_to_num(y.float())) for x, y in zip(a, b))


def test_results_that_overlap_what_is_read_are_refused():
    from multimodalsum_amd import kernels as kn
    buf = torch.zeros(20, 8, device="cuda")
    ids = torch.tensor([1, 2], device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        kn.embed_bwd(buf[9:11], ids, 10, out=buf[:10])
    assert torch.equal(kn.embed_bwd(buf[10:12] + 1, ids, 10, out=buf[:10])[:4, 0].cpu(), torch.tensor([0.0, 1.0, 1.0, 0.0]))
    out = kn.embed_bwd(buf[10:12], ids, 10, out=buf[:10], accumulate=True)
    assert out.data_ptr() == buf.data_ptr() and out.sum() == 16


@pytest.mark.parametrize("V,D,n", [(3, 1, 2048), (5, 7, 2047), (4200000, 2, 300), (1100000, 1030, 9), (64, 2050, 1000), (9, 512, 255), (2, 64, 2048)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_embedding_gradient_of_few_ids(V, D, n, accumulate):
    """Tables of one row a workgroup to millions; one id many times; the last rows of the table."""
    from multimodalsum_amd import kernels as kn
    g = torch.Generator().manual_seed(V + n)
    ids = torch.randint(max(V - 40, 0), V, (n,), generator=g)
    ids[: n // 3] = V - 1
    ids[n // 3] = -7
    ids = ids.cuda()
    dy = torch.randn(n, D, generator=g).cuda()
    rows, at = torch.unique(ids[ids >= 0], return_inverse=True)
    want = torch.zeros(len(rows), D, dtype=torch.float64, device="cuda").index_add_(0, at, 0.5 * dy[ids >= 0].double())
    mag = torch.zeros_like(want).index_add_(0, at, 0.5 * dy[ids >= 0].double().abs())
    out = torch.full((V, D), 3.0 if accumulate else float("nan"), device="cuda")
    got = kn.embed_bwd(dy, ids, V, 0.5, out=out, accumulate=accumulate)
    base = 3.0 if accumulate else 0.0
    assert ((got[rows].double() - want - base).abs() <= (mag * (n + 2) + 4 * abs(base)) * H).all()      # at most n additions in a row
    got.index_fill_(0, rows, base)
    assert (got == base).all()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n", [2049, 8193, 16384, 16385, 20001, 32768, 32769, 70000])
def test_embedding_gradient_of_skewed_ids(n, dt):
    """A text's frequencies: tokens of one position, of a stretch's length, over hundreds of stretches; padding in front and behind."""
    from multimodalsum_amd import kernels as kn
    V, D = 5003, 136
    g = torch.Generator().manual_seed(n)
    ids = torch.multinomial(1.0 / torch.arange(1, V + 1).double() ** 1.1, n, True, generator=g).cuda()
    dy = torch.randn(n, D, generator=g).to(dt).cuda()
    keep = ids != 1
    want, mag = torch.zeros(V, D, dtype=torch.float64, device="cuda"), torch.zeros(V, D, dtype=torch.float64, device="cuda")
    want.index_add_(0, ids[keep], 1.5 * dy[keep].double())
    mag.index_add_(0, ids[keep], 1.5 * dy[keep].double().abs())
    got = kn.embed_bwd(dy, ids, V, 1.5, 1)
    deep = torch.bincount(ids, minlength=V)[:, None].double() + 2       # additions into one sum, the scale
    assert ((got.double() - want).abs() <= mag * deep * H).all()
    assert torch.equal(got, kn.embed_bwd(dy, ids, V, 1.5, 1))


@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("P,T", [(1, 156), (3, 700), (40, 64), (300, 256), (1, 5000)])
def test_margins_of_long_sequences_keep_their_digits(P, T, average):
    """Sums of hundreds whose difference is small: the margin is the 64-bit sum of the tokens' values rounded once, by both forms of the loss."""
    from multimodalsum_amd import kernels as kn
    g = torch.Generator().manual_seed(P * T)
    V = 11
    labels = torch.randint(0, V, (2 * P, T), generator=g)
    labels[:, -3:] = -100
    logp = -torch.rand(2 * P, T, generator=g) * 4
    ref = logp.masked_fill(labels < 0, 0.0).sum(1) / (T - 3 if average else 1) + torch.randn(2 * P, generator=g) * 1e-3
    keep = (labels >= 0).double()
    S = (logp.double() * keep).sum(1) / (T - 3 if average else 1)
    r = S - ref.double()
    h = 0.5 * (r[:P] - r[P:])
    loss, margins, seq, coef = kn.preference_pairs(logp.cuda(), labels.cuda(), ref.cuda(), V, 0.5, 0.1, average)
    assert ((margins.cpu().double() - h).abs() <= 2 * H * h.abs() + 2.0 ** -40).all()       # 64-bit sums of up to 5,000 values below 4: 2^-53 of them a step
    assert ((seq.cpu().double() - S).abs() <= 2 * H * S.abs()).all()
    x = torch.randn(2 * P, T, V, generator=g).cuda()
    lp = kn.token_logprob(x, labels.cuda())
    want = kn.preference_pairs(lp, labels.cuda(), ref.cuda(), V, 0.5, 0.1, average)
    got = kn.preference_loss(x, labels.cuda(), ref.cuda(), 0.5, 0.1, average)
    for a, b in zip(want[:3], got[:3]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("N,T", [(4, 64), (16, 512), (64, 1024)])
def test_policy_loss_of_terms_that_cancel(N, T):
    from multimodalsum_amd import kernels as kn
    g = torch.Generator().manual_seed(N)
    adv = torch.randn(N, T, generator=g)
    adv -= adv.mean()
    logp = -torch.rand(N, T, generator=g)
    out, coef = kn.policy_terms(logp.cuda(), torch.zeros(N, T, dtype=torch.int64).cuda(), logp.cuda(), adv.cuda(), None, 5, 0.2, 0.2, 0.0, "token")
    want = -adv.double().mean()                                     # ratios of one, weights a power of two: every term is exact
    assert abs(out[0].item() - want) <= 2 * H * abs(want) + 2.0 ** -50
    assert torch.equal(coef.cpu(), -adv / (N * T))
