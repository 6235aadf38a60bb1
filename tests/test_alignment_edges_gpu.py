"""GPU: the scoring / loss / embedding / 8-bit operators at the edges of what their entry points take."""
import pytest
import torch

pytestmark = pytest.mark.gpu
H = 2.0 ** -24                       # half a step of f32


@pytest.mark.parametrize("n", [40, 3000])
@pytest.mark.parametrize("pad", [-1, -2, -50, 0])
def test_padding_rows_counted_from_the_end(pad, n):
    """The padding row stays zero under a step, by the one-launch gradient and by the sorted one."""
    import multimodalsum_amd as mm
    ids = (torch.arange(n, device="cuda") * 7) % 50
    m = mm.ScaledEmbedding(50, 16, scale=2.0, padding_idx=pad)
    y = m(ids)
    assert (y[ids == pad % 50] == 0).all()
    y.sum().backward()
    want = 2.0 * torch.bincount(ids, minlength=50).float()
    want[pad] = 0.0
    assert torch.equal(m.weight.grad, want[:, None].expand(50, 16))
    assert torch.equal(mm.scaled_embedding_grad(torch.ones(n, 16, device="cuda"), ids, 50, 2.0, padding_idx=pad), m.weight.grad)


def test_losses_may_be_changed_in_place():
    """Accumulation steps: loss /= 4 and a change of what is kept for monitoring, then the backward pass."""
    import multimodalsum_amd as mm
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 5, 50, generator=g).cuda()
    labels, adv = torch.randint(0, 50, (6, 5), generator=g).cuda(), torch.randn(6, generator=g).cuda()
    _, old = mm.sequence_logprobs(x, labels)
    pref, pol = mm.PreferenceLoss(beta=0.3), mm.ClippedPolicyLoss(kl_coef=0.1)
    for call, kept in ((lambda t: pref(t, labels), lambda: (pref.margins, pref.logps)), (lambda t: pol(t, labels, old - 0.1, adv, old + 0.2), lambda: (pol.kl, pol.clipped, pol.logps))):
        a, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
        call(a).backward()
        loss = call(b)
        loss /= 4
        for t in kept():
            t.zero_()
        loss.backward()
        assert torch.equal(b.grad, a.grad / 4) and (a.grad != 0).any()      # a power of two: exact


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_sums_of_exponentials_are_not_biased(dt):
    """Sums of exponentials are off by rounding (H of a term's argument times its size, H of the exponential and of every addition), in either
    direction: over 2,048 rows the average is a 45th of it.  A third of H bounds what may share a sign (a factor log2 e in one f32 word: 1.04 H)."""
    from multimodalsum_amd import kernels as kn
    g = torch.Generator(device="cuda").manual_seed(4)
    for V in (50265, 110003):                                        # a row in registers; a row read in steps
        off = []
        for _ in range(16):
            x = (torch.randn(1, 128, V, generator=g, device="cuda") * 2).to(dt)
            stats = torch.empty(1, 128, 2, device="cuda")
            kn.token_logprob(x, torch.zeros(1, 128, dtype=torch.int64, device="cuda"), stats)
            s = (x.double() - x.double().amax(-1, keepdim=True)).exp().sum(-1)
            off.append(stats[..., 1].double() / s - 1)
        off = torch.stack(off)
        assert off.mean().abs() < H / 3 and off.abs().max() < 160 * H


@pytest.mark.parametrize("M", [1, 40, 400, 40000])
def test_gelu_of_the_8bit_linear_layer(M):
    """The epilogue's GELU by itself: activations of one give y = w's row, at every size of x; from the tail to values that pass through, zero and infinities.

    Bounds, relative, from the argument z as the same product without GELU has it: the polynomials and their products 10 H, the exponential's argument
    z^2 / 2 rounded twice (and its factor) 3 z^2 H at most; bf16: the fit's 2.4e-5 and half a step of the result on top.  Results below 1e-37 are zero."""
    from multimodalsum_amd import kernels as kn
    w = torch.cat([torch.linspace(-13, 13, 2001), torch.linspace(-1.2, 1.2, 1001), torch.logspace(-30, 30, 301), -torch.logspace(-30, 0, 301), torch.zeros(1)])
    N = w.numel()
    qx, sx = kn.quantize_rows(torch.ones(M, 8, device="cuda"))
    qw, sw = kn.quantize_rows(torch.full((N, 8), 1.0, device="cuda"))
    qx[:, 1:] = 0                                                     # one product of 127 127
    bias = w.cuda() - (127.0 * 127.0 * sx[0] * sw)                   # y = one product + bias
    y = torch.addcmul(bias.double(), torch.full((), 127.0 * 127.0, dtype=torch.float64, device="cuda"), sx[0].double() * sw.double())
    for out in (torch.float32, torch.bfloat16):
        got = kn.gemm_i8(qx, sx, qw, sw, torch.empty(M, N, dtype=out, device="cuda"), bias, True)
        assert (got == got[0]).all()
        plainly = kn.gemm_i8(qx, sx, qw, sw, torch.empty(M, N, device="cuda"), bias, False)[0].double()      # the argument as the epilogue has it
        assert ((plainly - y).abs() <= 4 * H * (1 + y.abs())).all()
        z = plainly
        want = z * 0.5 * torch.special.erfc(-z / 2 ** 0.5)
        rel = H * (10 + 3 * z * z) if out == torch.float32 else 2.4e-5 + H * (10 + 4 * z * z) + torch.finfo(out).eps / 2
        assert ((got[0].double() - want).abs() <= rel * want.abs() + 1e-37).all(), (((got[0].double() - want).abs()) / (rel * want.abs() + 1e-37)).max().item()
        edge = torch.tensor([float("inf"), float("-inf"), float("nan"), 3e38, -3e38], device="cuda")
        got = kn.gemm_i8(qx, sx, qw[:5], sw[:5], torch.empty(M, 5, dtype=out, device="cuda"), edge, True)[M - 1]
        assert got[0] == float("inf") and got[1] == 0 and torch.isnan(got[2]) and got[3] > 2.9e38 and got[4] == 0


def test_kl_estimate_and_its_gradient_near_zero():
    """d = ref - logp from 1e-7 to 30, both signs: e^d - d - 1 and 1 - e^d keep their digits (an f32 difference of e^d and 1 has none left at 1e-7).

    d is rounded once (H; exact below 2^-24 of its parts), d^2 / 2 doubles that; the series or e^d - 1 and a difference from 1/2 on, where the result is
    a quarter of its parts: 16 H in all; beyond 1, d e^d / (e^d - 1) H more for d's own rounding."""
    from multimodalsum_amd import kernels as kn
    size = torch.logspace(-7, 1.4, 500)
    d = torch.cat([size, -size, torch.tensor([0.0, 0.5, -0.5])])
    N = d.numel()
    labels, adv = torch.zeros(N, 1, dtype=torch.int64, device="cuda"), torch.zeros(N, device="cuda")
    ref = d.cuda().view(N, 1)
    logp = torch.zeros(N, 1, device="cuda")                           # d is ref itself
    out, coef = kn.policy_terms(logp, labels, logp, adv, ref, 5, 0.2, 0.2, 1.0, "sequence")
    g = ref.double().view(-1)
    want = -torch.expm1(g) / N
    assert ((coef.double().view(-1) - want).abs() <= (16 + 2 * g.abs()) * H * want.abs()).all()
    for i in range(0, N, 10):                                          # the estimates one by one
        out, _ = kn.policy_terms(logp[:1], labels[:1], logp[:1], adv[:1], ref[i:i + 1], 5, 0.2, 0.2, 0.5, "sequence")
        z = g[i].item()
        kl = torch.expm1(g[i]).item() - z if abs(z) > 1e-2 else z * z / 2 + z ** 3 / 6 + z ** 4 / 24 + z ** 5 / 120 + z ** 6 / 720
        assert abs(out[1].item() - kl) <= (16 + 2 * abs(z)) * H * kl and abs(out[0].item() - 0.5 * kl) <= (18 + 2 * abs(z)) * H * kl, (z, out[1].item(), kl)


def test_kl_without_a_coefficient_is_only_reported():
    """kl_coef = 0 with a reference that disagrees by more than e^88 on a token: the estimate is infinite, loss and gradient do not know of it."""
    import multimodalsum_amd as mm
    x = torch.randn(2, 3, 40, generator=torch.Generator().manual_seed(0)).cuda()
    labels, adv = torch.zeros(2, 3, dtype=torch.int64, device="cuda"), torch.tensor([1.0, -1.0], device="cuda")
    x[0, 1, 0] = -300.0
    old = mm.sequence_logprobs(x, labels)[1] - 0.1
    ref = old.clone()
    ref[0, 1], ref[1, 2] = -1.0, float("-inf")
    plain = mm.policy_loss_and_grad(x, labels, old, adv)
    got = mm.policy_loss_and_grad(x, labels, old, adv, ref)
    assert torch.equal(got[0], plain[0]) and torch.equal(got[4], plain[4]) and got[1] == float("inf") and torch.isfinite(got[4]).all()
    xg = x.clone().requires_grad_(True)
    loss = mm.ClippedPolicyLoss()(xg, labels, old, adv, ref)
    loss.backward()
    assert torch.isfinite(loss) and torch.isfinite(xg.grad).all()


def test_more_rows_than_a_grid_axis_holds():
    """2^26 rows and a few: an axis of a launch holds fewer than 2^32 threads, 2^26 workgroups of one wave, 2^24 of four."""
    import multimodalsum_amd as mm
    N, T, V = 2 ** 25 + 6, 2, 2
    x = torch.zeros(N, T, V, dtype=torch.bfloat16, device="cuda")
    labels = torch.zeros(N, T, dtype=torch.int64, device="cuda")
    x[-1, 1, 0], x[-3, 0, 0], x[5, 0, 0] = 2.0, -1.0, 3.0
    labels[-2] = -100
    probe = torch.tensor([0, 5, N // 2, N - 3, N - 2, N - 1], device="cuda")
    lp = torch.log_softmax(x[probe].double(), -1)[..., 0] * (labels[probe] >= 0)
    seq, tok = mm.sequence_logprobs(x, labels)
    for got, want in ((tok[probe], lp), (seq[probe], lp.sum(1))):
        assert ((got.double() - want).abs() <= 8 * H).all()
    half = torch.tensor(0.5, dtype=torch.float64).log().item()
    assert (tok[6:N - 3] - half).abs().max() <= 8 * H and (seq[6:N - 3] - 2 * half).abs().max() <= 16 * H
    P = N // 2
    loss, margins, d = mm.preference_loss_and_grad(x, labels, beta=0.5)
    c = (torch.sigmoid(-margins.double()) * 0.5 / P)[torch.arange(N, device="cuda") % P]      # -d loss / d log p of the chosen one
    c[P:] *= -1
    assert (margins[6:P - 3] == 0).all() and (loss.double() - torch.nn.functional.softplus(-margins.double()).mean()).abs() <= 8 * H
    p1 = torch.softmax(x.double(), -1)[..., 1] * (labels >= 0)
    want = torch.stack([-c[:, None] * p1, c[:, None] * p1], -1)
    assert ((d.double() - want).abs() <= want.abs() * 2.0 ** -8 * 1.01).all()
    old, adv = tok, torch.ones(N, device="cuda")
    for reduction in ("token", "sequence"):
        l, _, _, tok2, d2 = mm.policy_loss_and_grad(x, labels, old, adv, reduction=reduction)
        assert torch.equal(tok2, tok)
        w = torch.full((N, 1), 1.0 / (2 * N - 2) if reduction == "token" else 0.5 / N, dtype=torch.float64, device="cuda")
        want = torch.stack([-w * p1, w * p1], -1)                   # d loss / d log p = -A w, and the label is 0
        assert ((d2.double() - want).abs() <= want.abs() * 2.0 ** -8 * 1.01).all()
        mean = (2 * N - 2) / (2 * N - 2) if reduction == "token" else (N - 1) / N
        assert abs(l.item() + mean) <= 4 * H


def test_more_ids_than_a_grid_axis_holds():
    import multimodalsum_amd as mm
    n, V, D = 2 ** 27 + 3, 1000, 129                                 # a workgroup takes eight of these rows
    table = (torch.arange(V, device="cuda")[:, None] * 0.25 + torch.arange(D, device="cuda") * 0.5).bfloat16()
    y = mm.scaled_embedding(torch.arange(n, device="cuda") % V, table, 2.0)
    assert torch.equal(y[:V], table * 2) and torch.equal(y[-V:], (table * 2).roll(-((n - V) % V), 0))
    for lo in range(0, n, 2 ** 24):
        k = min(n, lo + 2 ** 24) - lo
        assert torch.equal(y[lo:lo + k, 77], (table[:, 77] * 2)[(torch.arange(k, device="cuda") + lo) % V])
    del y
    torch.cuda.empty_cache()
    n, V = 2 ** 29 + 5, 4099                                         # 2^24 stretches of 32 sorted positions
    ids = torch.arange(n, device="cuda") % V
    got = mm.scaled_embedding_grad(torch.ones(n, 1, dtype=torch.bfloat16, device="cuda"), ids, V, 0.5, padding_idx=7)
    want = torch.bincount(ids, minlength=V).float() * 0.5            # below 2^24: exact in any order
    want[7] = 0.0
    assert torch.equal(got[:, 0], want)
    del ids
    torch.cuda.empty_cache()


def test_more_tokens_to_quantise_than_a_grid_axis_holds():
    from multimodalsum_amd import kernels as kn
    M = 2 ** 26 + 5
    x = torch.ones(M, 2, device="cuda")
    x[:, 1] = torch.arange(M, device="cuda") % 101 * 0.01
    q, s = kn.quantize_rows(x)
    assert (q[:, 0] == 127).all() and torch.equal(s, torch.full_like(s, 1.0) / 127.0)
    for lo in range(0, M, 2 ** 24):
        assert torch.equal(q[lo:lo + 2 ** 24, 1].float(), torch.round(x[lo:lo + 2 ** 24, 1].double() * 127).float())
    assert not q[-1000:, 2:].any() and not q[:1000, 2:].any()
    del q, x
    torch.cuda.empty_cache()


def test_int8_layer_in_a_model_that_is_cast():
    import multimodalsum_amd as mm
    lin = mm.Int8Linear(torch.randn(40, 24, device="cuda"), torch.randn(40, device="cuda"), out_dtype=torch.float32)
    x = torch.randn(5, 24, device="cuda").bfloat16()
    want = lin(x)
    model = torch.nn.Sequential(torch.nn.Linear(24, 24, device="cuda"), lin).bfloat16()
    assert model[0].weight.dtype == torch.bfloat16 and torch.equal(model[1](x), want)


# up to 64 rows into many columns: workgroups of 64 columns, the last one not full, for one, two and four blocks of 16 rows
I8_WIDE = [(1, 32769, 256), (16, 50265, 1024), (17, 16385, 384), (32, 50265, 1024), (33, 16400, 300), (64, 20011, 512)]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", I8_WIDE)
def test_int8_linear_of_few_rows_into_many_columns(M, N, K, dt):
    """Exact integer sums in 64 bits; the sum's conversion, two scales and the bias: 8 H of the parts, GELU as for the other sizes 40 H, half a step of the result."""
    from multimodalsum_amd import Int8Linear, _lib, kernels as kn
    g = torch.Generator().manual_seed(M + N + K)
    x = (torch.randn(M, K, generator=g) * (0.2 + torch.rand(M, 1, generator=g))).to(dt).cuda()
    lin = Int8Linear((torch.randn(N, K, generator=g) * 0.05).cuda(), torch.randn(N, generator=g).cuda())
    assert kn.linear_i8_plan(M, N, K)[:3] == (_lib.I8_PLAN_FEW, 16 if M <= 16 else 32 if M <= 32 else 64, 64)
    qx, sx = kn.quantize_rows(x)
    product = torch.mm(qx.double(), lin.qweight.double().t().contiguous()) * sx.double()[:, None] * lin.scale.double()
    for bias, gelu in ((None, False), (lin.bias, False), (lin.bias, True)):
        want = product if bias is None else product + bias.double()
        mag = product.abs() + (0.0 if bias is None else bias.double().abs())
        if gelu:
            want = 0.5 * want * torch.special.erfc(-want / 2 ** 0.5)
        for out in (torch.float32, torch.bfloat16):
            wide = torch.full((M + 2, N + 6), float("nan"), dtype=out, device="cuda")
            kn.linear_i8(x, lin.qweight, lin.scale, wide[1:-1, 3:N + 3], bias, gelu)
            y = wide[1:-1, 3:N + 3].double()
            assert ((y - want).abs() <= mag * (40 if gelu else 8) * H + want.abs() * torch.finfo(out).eps / 2 + torch.finfo(out).tiny).all()
            assert torch.isnan(wide[0]).all() and torch.isnan(wide[-1]).all() and torch.isnan(wide[:, :3]).all() and torch.isnan(wide[:, N + 3:]).all()


@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("eps", [0.0, 0.1])
@pytest.mark.parametrize("P,T,V", [(1, 1100, 5), (16, 300, 7), (17, 300, 7), (33, 1000, 3), (300, 40, 9)])
def test_preference_gradient_of_long_sequences(P, T, V, eps, average):
    """The factor of every sequence and the gradient of the logits, by both forms, against 64 bits from the f32 log-probabilities that the kernel itself
    sums, so that only these roundings count.  h: the f32 of a 64-bit sum (beta and ref are f32 values): H |h|.  Factor: sigmoid's slope in h is below its
    value, so |h| H, and the exponential, quotient, difference (smoothing: of values it is a tenth of at least) and four products: 40 H in all.  Gradient:
    the row's own statistics on top, 400 H of the factor's two products for rows of this kind.  What the tolerance rejects is asserted beside it."""
    from multimodalsum_amd import kernels as kn
    g = torch.Generator().manual_seed(P + T)
    x = torch.randn(2 * P, T, V, generator=g).cuda()
    labels = torch.randint(0, V, (2 * P, T), generator=g)
    for i in range(2 * P):                                             # ragged, one sequence empty
        labels[i, T - (7 * i) % (T // 2):] = -100
    if P > 1:
        labels[1] = -100
    labels = labels.cuda()
    keep = (labels >= 0) & (labels < V)
    stats = torch.empty(2 * P, T, 2, device="cuda")
    logp = kn.token_logprob(x, labels, stats)
    cnt = keep.sum(1).clamp(min=1).double()
    seq = (logp.double() * keep).sum(1) / (cnt if average else 1.0)
    ref = (seq + torch.randn(2 * P, generator=g).cuda() * 2).float()    # margins of a few units
    beta = torch.tensor(0.3).item()
    r = seq - ref.double()
    h = beta * (r[:P] - r[P:])
    dh = (eps - torch.sigmoid(-h)) * beta / P
    want = torch.cat([dh, -dh]) / (cnt if average else 1.0)
    loss, margins, got_seq, coef = kn.preference_pairs(logp, labels, ref, V, 0.3, eps, average)
    tol = (40 + 2 * h.abs().repeat(2)) * H * torch.cat([beta / P * (eps + torch.sigmoid(-h))] * 2) / (cnt if average else 1.0)
    assert ((coef.double() - want).abs() <= tol).all() and (tol < 0.01 * want.abs().max()).all()
    p = torch.softmax(x.double(), -1)
    lab = torch.where(keep, labels, torch.zeros_like(labels))
    one = torch.zeros_like(p).scatter_(-1, lab[..., None], 1.0)
    d_want = torch.where(keep[..., None], want[:, None, None] * (one - p), torch.zeros_like(p))
    d_tol = (tol[:, None, None] + 400 * H * want.abs()[:, None, None]) * (one + p)
    fused = kn.preference_loss(x, labels, ref, 0.3, eps, average)
    assert torch.equal(fused[0], loss) and torch.equal(fused[1], margins) and torch.equal(fused[2], got_seq)
    for d in (fused[3], kn.token_logprob_bwd(x, labels, stats, coef)):
        assert ((d.double() - d_want).abs() <= d_tol).all() and (d[~keep] == 0).all()
    for wrong in (torch.zeros_like(d_want), -d_want, 2 * d_want, d_want.roll(1, 0)) + ((d_want * cnt[:, None, None],) if average else ()):
        assert not ((wrong - d_want).abs() <= d_tol).all()


def test_gradient_over_the_padded_buffer_of_one_row():
    import multimodalsum_amd as mm
    for dt in (torch.float32, torch.bfloat16):
        for V in (50, 50265, 110003):
            buf = torch.randn(1, 1, V + 7, generator=torch.Generator().manual_seed(V)).to(dt).cuda()
            args = (torch.full((1, 1), 3, device="cuda"), torch.full((1, 1), -2.0, device="cuda"), torch.ones(1, device="cuda"))
            want = mm.policy_loss_and_grad(buf[:, :, :V].clone(), *args)
            got = mm.policy_loss_and_grad(buf[:, :, :V], *args, dlogits=buf)
            assert torch.equal(got[0], want[0]) and torch.equal(buf[:, :, :V], want[4]) and (buf[:, :, V:] == 0).all()


@pytest.mark.parametrize("dt,P,T", [(torch.bfloat16, 16, 160), (torch.float32, 8, 160), (torch.bfloat16, 16, 141)])
def test_preference_loss_of_more_logits_than_the_cache_holds(dt, P, T):
    """Rows on both sides of the 400 MB that are left to the second reading: the fused call's numbers are the two-step form's, bit for bit, also over the
    logits themselves."""
    from multimodalsum_amd import kernels as kn
    V = 50265
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(2 * P, T, V, generator=g, device="cuda").to(dt)
    assert x.numel() * x.element_size() > 420 * 2 ** 20
    labels = torch.randint(0, V, (2 * P, T), generator=g, device="cuda")
    labels[3, 5:] = -100
    stats = torch.empty(2 * P, T, 2, device="cuda")
    logp = kn.token_logprob(x, labels, stats)
    loss, margins, seq, coef = kn.preference_pairs(logp, labels, None, V, 0.1, 0.0, False)
    want = kn.token_logprob_bwd(x, labels, stats, coef)
    for over in (None, x):
        got = kn.preference_loss(x, labels, None, 0.1, 0.0, False, over)
        for a, b in zip(got, (loss, margins, seq, want)):
            assert torch.equal(a, b)
    assert (want != 0).any() and not (want[3, 5:] != 0).any()
