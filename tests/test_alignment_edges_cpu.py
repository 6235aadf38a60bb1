"""CPU: calls of the scoring / loss / embedding / 8-bit entry points that have to be refused, and what the host does around a launch."""
import pytest
import torch

BF, F32 = 1, 0
FAKE = 1 << 20                       # a 16-byte aligned address: refused calls never dereference it


def refused(exc, fn, *a, **k):
    with pytest.raises(exc):
        fn(*a, **k)


def calls():
    """Every C entry with arguments that pass its checks (but for the launch, which needs a device): name, arguments, the positions of pointers that
    may be missing."""
    F = FAKE
    return [
        ("mmsum_token_logprob", [BF, F, 8, F, F, None, 4, 8, None], {5, 8}),
        ("mmsum_token_logprob_bwd", [BF, F, 8, F, F, F, 1, None, F, 8, 8, 4, 8, None], {7, 13}),
        ("mmsum_sequence_logprob", [F, F, 2, 3, 8, 0, F, None], {7}),
        ("mmsum_preference_pairs", [F, F, None, 2, 3, 8, 0.1, 0.0, 0, F, F, F, F, F, None], {2, 14}),
        ("mmsum_preference_loss", [BF, F, 8, F, None, 2, 3, 8, 0.1, 0.0, 0, F, F, F, F, 8, 8, F, None], {4, 17, 18}),
        ("mmsum_policy_terms", [F, F, F, None, F, 0, 2, 3, 8, 0.2, 0.2, 0.0, 0, F, F, F, None], {3, 15, 16}),
        ("mmsum_policy_loss", [BF, F, 8, F, F, None, F, 0, 2, 3, 8, 0.2, 0.2, 0.0, 0, F, F, F, 8, 8, F, None], {5, 20, 21}),
        ("mmsum_embed_fwd", [BF, F, F, 8, F, 8, 4, 10, 8, 1.0, None], {10}),
        ("mmsum_embed_bwd", [BF, F, 8, F, 4, 10, 8, 1.0, -1, 0, F, None, None], {11, 12}),
        ("mmsum_quantize_i8", [BF, F, 8, 4, 8, F, 128, F, None], {8}),
        ("mmsum_gemm_i8", [F, 128, F, F, 128, F, None, BF, F, 16, 4, 16, 128, 0, None], {6, 14}),
        ("mmsum_linear_i8", [BF, F, 128, F, 128, F, None, BF, F, 16, 4, 16, 128, 0, F, None], {6, 14, 15}),
    ]


@pytest.mark.parametrize("call", calls(), ids=lambda c: c[0])
def test_a_missing_pointer_is_refused(call):
    from multimodalsum_amd import _lib
    name, args, may_miss = call
    tried = 0
    for i, a in enumerate(args):
        if a == FAKE and i not in may_miss:
            assert getattr(_lib.lib, name)(*args[:i], None, *args[i + 1:]) == -3, (name, i)
            tried += 1
    assert tried >= 3


def test_missing_tensors_are_refused():
    import multimodalsum_amd as mm
    from multimodalsum_amd import kernels as kn
    x, lab, z, adv = torch.zeros(4, 3, 8), torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3), torch.zeros(4)
    refused(TypeError, mm.policy_loss_and_grad, x, lab, None, adv)
    refused(TypeError, mm.policy_loss_and_grad, x, lab, z, None)
    refused(TypeError, mm.policy_loss_and_grad, x, lab, z, 1.0)
    refused(TypeError, kn.policy_terms, z, lab, None, adv, None, 8, 0.2, 0.2, 0.0, "token")
    refused(ValueError, mm.policy_loss_and_grad, x, lab, z, torch.zeros(()))
    q, s, w = torch.zeros(4, 128, dtype=torch.int8), torch.zeros(4), torch.zeros(4, 128)
    refused(TypeError, kn.gemm_i8, q, None, q, s, torch.zeros(4, 4))
    refused(TypeError, kn.gemm_i8, q, s, q, None, torch.zeros(4, 4))
    refused(TypeError, kn.linear_i8, w, q, None)


class Recorder:
    """In place of a launch: what would have been launched; tensors stay on the CPU."""

    def __init__(self, monkeypatch, fill=None):
        from multimodalsum_amd import kernels as kn
        self.calls, self.fill = [], fill or {}
        monkeypatch.setattr(kn, "_device", lambda *t: torch.device("cpu"))
        monkeypatch.setattr(kn, "_p", lambda t: t)
        monkeypatch.setattr(kn, "_launch", self.launch)

    def launch(self, name, device, *args):
        self.calls.append((name, args))
        if name in self.fill:
            self.fill[name](*args)


def test_padding_rows_count_from_the_end(monkeypatch):
    import multimodalsum_amd as mm
    ids, dy = torch.tensor([[1, 9, 8]]), torch.ones(1, 3, 8)

    def written(*a):
        a[10].zero_()
    rec = Recorder(monkeypatch, {"mmsum_embed_bwd": written, "mmsum_embed_fwd": lambda *a: a[4].zero_()})
    for pad, row in ((None, -1), (0, 0), (1, 1), (9, 9), (-1, 9), (-2, 8), (-10, 0)):
        mm.scaled_embedding_grad(dy, ids, 10, padding_idx=pad)
        assert rec.calls[-1][0] == "mmsum_embed_bwd" and rec.calls[-1][1][8] == row
        t = torch.zeros(10, 8, requires_grad=True)
        mm.scaled_embedding(ids, t, 2.0, pad).sum().backward()
        assert rec.calls[-1][0] == "mmsum_embed_bwd" and rec.calls[-1][1][8] == row
        m = mm.ScaledEmbedding(10, 8, padding_idx=pad, device="cpu")
        assert (m.weight[row] == 0).all() if pad is not None else (m.weight != 0).any(1).all()
        m(ids).sum().backward()
        assert rec.calls[-1][0] == "mmsum_embed_bwd" and rec.calls[-1][1][8] == row
    for pad in (10, -11, 2 ** 40):
        refused(ValueError, mm.scaled_embedding_grad, dy, ids, 10, padding_idx=pad)
        refused(ValueError, mm.scaled_embedding, ids, torch.zeros(10, 8), 1.0, pad)
        refused(ValueError, mm.scaled_embedding, ids, torch.zeros(10, 8, requires_grad=True), 1.0, pad)
        refused(ValueError, mm.ScaledEmbedding, 10, 8, padding_idx=pad, device="cpu")
    refused(TypeError, mm.scaled_embedding_grad, dy, ids, 10, padding_idx=1.5)


def test_forward_mode_tangents_are_refused(monkeypatch):
    import torch.autograd.forward_ad as fwd
    import multimodalsum_amd as mm
    rec = Recorder(monkeypatch)
    lin = mm.Int8Linear(torch.ones(4, 8))
    ids, lab, z, adv = torch.tensor([1, 2]), torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3), torch.zeros(4)
    del rec.calls[:]
    with fwd.dual_level():
        for leaf in (False, True):
            table, x, logits = (fwd.make_dual(torch.ones(*s).requires_grad_(leaf), torch.ones(*s)) for s in ((10, 8), (3, 8), (4, 3, 8)))
            refused(RuntimeError, mm.scaled_embedding, ids, table, 2.0)
            refused(RuntimeError, lin, x)
            with torch.no_grad():
                refused(RuntimeError, lin, x)
            refused(RuntimeError, mm.PreferenceLoss(), logits, lab)
            refused(RuntimeError, mm.ClippedPolicyLoss(), logits, lab, z, adv)
    assert not [c for c in rec.calls if c[0] in ("mmsum_embed_fwd", "mmsum_linear_i8")]
    mm.scaled_embedding(ids, torch.ones(10, 8), 2.0)
    lin(torch.ones(3, 8))
    assert [c[0] for c in rec.calls][-2:] == ["mmsum_embed_fwd", "mmsum_linear_i8"]


@pytest.mark.parametrize("kind", ["preference", "policy"])
def test_losses_may_be_changed_in_place(monkeypatch, kind):
    """loss /= steps, loss += another loss, and changes of what the module keeps for monitoring leave the backward pass as it was."""
    import multimodalsum_amd as mm

    def fill(value, *at):
        def f(*a):
            for i in at:
                a[i].fill_(value)
        return f
    rec = Recorder(monkeypatch, {"mmsum_preference_pairs": fill(8.0, 9, 10, 11, 12, 13), "mmsum_policy_terms": fill(8.0, 13, 14),
                                 "mmsum_token_logprob_bwd": lambda *a: a[8].copy_(a[7] * a[5].reshape(-1)[0])})
    lab, z, adv = torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3), torch.zeros(4)
    for change in (lambda m, l: l.div_(4), lambda m, l: l.add_(torch.ones(())).div_(4), lambda m, l: (m.logps.zero_(), l.div_(4)),
                   lambda m, l: ((m.margins if kind == "preference" else m.kl).clamp_(max=1.0), l.div_(4)), lambda m, l: (l.detach().zero_(), l.div_(4))):
        x = torch.zeros(4, 3, 8, requires_grad=True)
        m = mm.PreferenceLoss() if kind == "preference" else mm.ClippedPolicyLoss()
        loss = m(x, lab) if kind == "preference" else m(x, lab, z, adv)
        assert loss.shape == () and loss == 8.0
        change(m, loss)
        loss.backward()
        assert (x.grad == 2.0).all() and rec.calls[-1][0] == "mmsum_token_logprob_bwd"


def test_results_written_into_a_tensor_count_as_changes_in_place(monkeypatch):
    """A backward pass that saved a tensor which a later call writes over raises instead of reading the gradient as logits."""
    import multimodalsum_amd as mm
    from multimodalsum_amd import kernels as kn
    Recorder(monkeypatch)
    lab, z, adv = torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3), torch.zeros(4)
    for fused in (lambda t: mm.preference_loss_and_grad(t, lab, dlogits=t), lambda t: mm.policy_loss_and_grad(t, lab, z, adv, dlogits=t),
                  lambda t: kn.token_logprob_bwd(t, lab, torch.zeros(4, 3, 2), z, dlogits=t)):
        for loss in (lambda t: mm.PreferenceLoss()(t, lab), lambda t: mm.ClippedPolicyLoss()(t, lab, z, adv), lambda t: (t * t).sum()):
            logits = torch.zeros(4, 3, 8, requires_grad=True) * 1.0
            value = loss(logits)
            with torch.no_grad():
                fused(logits)
            refused(RuntimeError, value.backward)
    q, s, out, stats, dy, ids = torch.zeros(4, 128, dtype=torch.int8), torch.zeros(4), torch.zeros(4, 4), torch.zeros(4, 3, 2), torch.zeros(3, 8), torch.tensor([1, 2, 3])
    for t, call in ((out, lambda t: kn.gemm_i8(q, s, q, s, t)), (out, lambda t: kn.linear_i8(torch.zeros(4, 128), q, s, t)), (stats, lambda t: kn.token_logprob(torch.zeros(4, 3, 8), lab, t)),
                    (torch.zeros(10, 8), lambda t: kn.embed_bwd(dy, ids, 10, out=t)), (torch.zeros(10, 8), lambda t: kn.embed_bwd(dy, ids, 10, out=t, accumulate=True)),
                    (torch.zeros(4, 3, 9), lambda t: mm.preference_loss_and_grad(torch.zeros(4, 3, 8), lab, dlogits=t))):
        before = t._version
        call(t)
        assert t._version > before
    with torch.inference_mode():                                   # tensors without a version
        t = torch.zeros(4, 3, 8)
        mm.preference_loss_and_grad(t, lab, dlogits=t)


def test_sizes_past_32_bits_are_refused():
    """Sizes that the C entries take as 32-bit numbers: ctypes would pass their lower halves."""
    import multimodalsum_amd as mm
    from multimodalsum_amd import kernels as kn

    def meta(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="meta")
    big = 2 ** 32 + 5
    lab1 = meta(2, 1, dtype=torch.int64)
    refused(ValueError, mm.sequence_logprobs, meta(2, 1, big), lab1)
    refused(ValueError, mm.sequence_logprobs, meta(big, 1, 5), meta(big, 1, dtype=torch.int64))
    refused(ValueError, mm.preference_loss_and_grad, meta(2, 1, 5), lab1, dlogits=meta(2, 1, big))
    refused(ValueError, kn.sequence_logprob, meta(2, 1), lab1, big)
    refused(ValueError, kn.sequence_logprob, meta(big, 1), meta(big, 1, dtype=torch.int64), 5)
    refused(ValueError, kn.preference_pairs, meta(2 * big, 1), meta(2 * big, 1, dtype=torch.int64), None, 5, 0.1, 0.0, False)
    refused(ValueError, kn.policy_terms, meta(big, 1), meta(big, 1, dtype=torch.int64), meta(big, 1), meta(big), None, 5, 0.2, 0.2, 0.0, "token")
    ids = meta(3, dtype=torch.int64)
    refused(ValueError, mm.scaled_embedding, ids, meta(big, 2))
    refused(ValueError, mm.scaled_embedding, ids, meta(2, big))
    refused(ValueError, mm.scaled_embedding_grad, meta(3, 2), ids, big)
    refused(ValueError, mm.scaled_embedding_grad, meta(3, big), ids, 2)
    refused(ValueError, kn.quantize_rows, meta(big, 2))
    q, s = meta(4, 128, dtype=torch.int8), meta(4)
    refused(ValueError, kn.gemm_i8, meta(big, 128, dtype=torch.int8), meta(big), q, s, meta(big, 4))
    refused(ValueError, kn.gemm_i8, q, s, meta(big, 128, dtype=torch.int8), meta(big), meta(4, big))
    refused(ValueError, kn.linear_i8, meta(big, 128), q, s)
    refused(ValueError, kn.linear_i8, meta(4, 128), meta(big, 128, dtype=torch.int8), meta(big))


def quantised(*a):
    """mmsum_quantize_i8 on the CPU."""
    x, M, K, q, scale = a[1].detach().double(), a[3], a[4], a[5], a[7]
    top = x.abs().amax(1)
    q.zero_()
    q[:, :K] = torch.nan_to_num(torch.round(x * 127 / top[:, None])).to(torch.int8)
    scale.copy_((top / 127).float())


def test_int8_layer_keeps_its_scales_under_casts(monkeypatch):
    """model.bfloat16(), .half(), .to(dtype), .double(): scales and bias stay f32, bit for bit; devices still move; the rest of the model is cast."""
    import multimodalsum_amd as mm
    rec = Recorder(monkeypatch, {"mmsum_quantize_i8": quantised})
    w, b = torch.randn(6, 8), torch.randn(6)
    for cast in (lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(), lambda m: m.to("cpu", torch.bfloat16), lambda m: m.float()):
        m = torch.nn.Sequential(torch.nn.Linear(3, 8), mm.Int8Linear(w, b))
        q, s = m[1].qweight.clone(), m[1].scale.clone()
        kind = cast(torch.nn.Linear(2, 2)).weight.dtype
        assert cast(m)[0].weight.dtype == kind
        assert m[1].scale.dtype == m[1].bias.dtype == torch.float32 and torch.equal(m[1].scale, s) and torch.equal(m[1].bias, b) and torch.equal(m[1].qweight, q)
        x = torch.zeros(2, 8, dtype=torch.bfloat16)
        assert m[1](x).dtype == torch.bfloat16 and rec.calls[-1][0] == "mmsum_linear_i8"
    m = mm.Int8Linear(w).bfloat16()
    assert m.bias is None and m.scale.dtype == torch.float32
    moved = mm.Int8Linear(w, b).to("meta")
    assert moved.scale.device.type == moved.bias.device.type == moved.qweight.device.type == "meta" and moved.scale.dtype == torch.float32
    back = moved.to_empty(device="cpu")
    assert back.scale.device.type == back.bias.device.type == "cpu" and back.scale.dtype == torch.float32


def test_int8_layer_from_its_state_dict(monkeypatch):
    """A saved layer without its float weights: a layer of the same sizes, made from zeros, loads it."""
    import multimodalsum_amd as mm
    Recorder(monkeypatch, {"mmsum_quantize_i8": quantised})
    for bias in (None, torch.randn(6)):
        saved = mm.Int8Linear(torch.randn(6, 8), bias).state_dict()
        again = mm.Int8Linear(torch.zeros(6, 8), None if bias is None else torch.zeros(6)).bfloat16()
        again.load_state_dict(saved)
        assert again.state_dict().keys() == saved.keys() and all(torch.equal(v, saved[k]) and v.dtype == saved[k].dtype for k, v in again.state_dict().items())


def test_int8_plan():
    """Every product of the 8-bit linear layer is reached by sizes that the GPU tests run; the rules' borders; the plan needs no device."""
    from multimodalsum_amd import _lib, kernels as kn
    from tests import test_alignment_edges_gpu as edges, test_alignment_ops_gpu as ops
    few, inside, ring, w4 = _lib.I8_PLAN_FEW, _lib.I8_PLAN_FEW_QUANTISING, _lib.I8_PLAN_RING, _lib.I8_PLAN_W4

    def p(M, N, K, **kw):
        return kn.linear_i8_plan(M, N, K, **kw)[:3]
    assert kn.linear_i8_plan(8, 1024, 1024) == (inside, 16, 16, 64) and p(9, 1024, 1024) == (few, 16, 16) and p(8, 1024, 1024, quantise=False) == (few, 16, 16)
    assert p(8, 16385, 1024) == (few, 16, 16) and p(16, 32768, 128) == (few, 16, 64) and p(17, 16383, 128) == (few, 32, 16) and p(17, 16384, 128) == (few, 32, 64)
    assert p(33, 100, 128) == (few, 64, 16) and p(64, 50265, 1024) == (few, 64, 64) and p(65, 50265, 1024) == (ring, 64, 64) == p(128, 4096, 1024)
    assert kn.linear_i8_plan(32, 50265, 1024) == (few, 32, 64, 786)
    assert p(36864, 4096, 1024) == (w4, 256, 256) and p(36864, 4096, 1024, gelu=True) == p(36864, 1024, 4096) == (ring, 192, 128) and kn.linear_i8_plan(8192, 8192, 8192) == (w4, 256, 256, 256)
    listed = ops.I8 + edges.I8_WIDE
    edge = [m.args[1] for m in ops.test_int8_product_at_tile_edges.pytestmark if m.name == "parametrize" and m.args[0] == "M,N,K"][0]
    for gelu in (False, True):
        reached = {p(M, N, K, gelu=gelu) for M, N, K in listed} | {p(M, N, -(-K // 128) * 128, gelu=gelu, quantise=False) for M, N, K in edge}
        assert reached == {(inside, 16, 16), (few, 16, 16), (few, 16, 64), (few, 32, 16), (few, 32, 64), (few, 64, 16), (few, 64, 64), (ring, 64, 64), (ring, 192, 128),
                           (w4, 256, 256)}, reached
        at_edges = [p(M, N, -(-K // 128) * 128, gelu=gelu, quantise=False) for M, N, K in edge]
        assert at_edges.count((w4, 256, 256)) >= 2 and at_edges.count((ring, 192, 128)) >= 2, at_edges
    for bad in ((0, 4, 128), (4, 0, 128), (4, 4, 0), (4, 4, 131073)):
        refused(RuntimeError, kn.linear_i8_plan, *bad)
    refused(RuntimeError, kn.linear_i8_plan, 4, 4, 100, quantise=False)
    for M, K in ((1, 1), (3, 128), (5, 129), (1000, 131072), (2 ** 20, 4096)):      # the entry's own statement of its workspace: rows padded to 128, then their scales
        assert _lib.lib.mmsum_linear_i8_workspace(M, K) == M * (-(-K // 128) * 128 + 4)


def test_the_build_checks_the_counted_wait(tmp_path):
    """The four-wave 8-bit kernel's vmcnt(40) counts on 32 wide stores in a row: the build's check accepts those and nothing else."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "multimodalsum_amd", "csrc", "check_handoff.py")
    spec = importlib.util.spec_from_file_location("check_handoff", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    store, wait = "\tglobal_store_dwordx4 v[0:1], v[2:5], off", "\ts_waitcnt vmcnt(40)"

    def rc(*lines):
        f = tmp_path / "k.s"
        f.write_text("\n".join(["_Z17gemm_i8_w4_kernelIDF16bLb1EEvX:", *lines, "\ts_endpgm", ".Lfunc_end0:"]) + "\n")
        return mod.main([str(f)])
    tail = ["\ts_cbranch_scc0 .LBB0_1", "\tglobal_store_short v0, v1, off"]
    assert rc(wait, *[store] * 32, *tail) == 0 and rc(*["\tv_add_f32 v0, v0, v1", store] * 32, wait, *tail) == 0
    assert rc(wait, *[store] * 31, *tail) == 1 and rc(wait, *[store] * 33, *tail) == 1 and rc(*[store] * 32, *tail) == 1
    assert rc(wait, *[store] * 16, "\ts_branch .LBB0_2", *[store] * 16) == 1 and rc(wait, *[store] * 16, "\tglobal_load_dword v0, v1, off", *[store] * 16) == 1
    assert rc("\ts_waitcnt vmcnt(41)", *[store] * 32) == 1


def test_gradient_over_the_padded_buffer_of_the_logits(monkeypatch):
    """dlogits = the buffer that the logits are a view of: for any number of rows, one among them; buffers of another pitch or start stay refused."""
    import multimodalsum_amd as mm
    rec = Recorder(monkeypatch)
    for N, T in ((4, 3), (2, 1), (1, 3), (1, 1)):
        lab, z, adv = torch.zeros(N, T, dtype=torch.int64), torch.zeros(N, T), torch.zeros(N)
        for W in (8, 9, 12):
            buf = torch.zeros(N, T, 12)
            assert mm.policy_loss_and_grad(buf[:, :, :8], lab, z, adv, dlogits=buf[:, :, :W])[4].data_ptr() == buf.data_ptr()
            assert rec.calls[-1][1][18:20] == (12 if N * T > 1 else W, W)
        for other in (buf[:, :, 1:9], buf[:, :, 4:]):
            refused(ValueError, mm.policy_loss_and_grad, buf[:, :, :8], lab, z, adv, dlogits=other)
    refused(ValueError, mm.policy_loss_and_grad, buf.view(-1)[:8].view(1, 1, 8).expand(1, 1, 8), torch.zeros(1, 1, dtype=torch.int64), torch.zeros(1, 1), torch.zeros(1),
            dlogits=buf.view(-1)[2:10].view(1, 1, 8))


def test_int8_layer_under_type(monkeypatch):
    """Module.type casts every buffer, the 8-bit weights among them: the layer keeps its own types."""
    import multimodalsum_amd as mm
    Recorder(monkeypatch, {"mmsum_quantize_i8": quantised})
    lin = mm.Int8Linear(torch.randn(6, 8), torch.randn(6))
    want = {k: v.clone() for k, v in lin.state_dict().items()}
    for dtype in (torch.bfloat16, torch.float64):
        got = lin.type(dtype).state_dict()
        assert all(torch.equal(got[k], v) and got[k].dtype == v.dtype for k, v in want.items())
