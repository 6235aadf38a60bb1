"""CPU: what the scoring / preference / policy / embedding / 8-bit entry points refuse, before anything touches a device."""
import pytest
import torch

BF = 1
FAKE = 1 << 20                       # a 16-byte aligned address: refused calls never dereference it


def test_c_entries_refuse():
    from multimodalsum_amd import _lib
    lib = _lib.lib
    lp = lib.mmsum_token_logprob
    assert lp(7, FAKE, 8, FAKE, FAKE, None, 4, 8, None) == -2
    assert lp(BF, FAKE, 7, FAKE, FAKE, None, 4, 8, None) == -1 and lp(BF, FAKE, 8, FAKE, FAKE, None, 0, 8, None) == -1 and lp(BF, FAKE, 8, FAKE, FAKE, None, 4, 0, None) == -1
    assert lp(BF, FAKE + 1, 8, FAKE, FAKE, None, 4, 8, None) == -3 and lp(0, FAKE + 2, 8, FAKE, FAKE, None, 4, 8, None) == -3
    bwd = lib.mmsum_token_logprob_bwd
    assert bwd(BF, FAKE, 8, FAKE, FAKE, FAKE, 0, None, FAKE, 8, 8, 4, 8, None) == -1                 # rows_per_coef
    assert bwd(BF, FAKE, 8, FAKE, FAKE, FAKE, 1, None, FAKE, 8, 7, 4, 8, None) == -1                 # W < V
    assert bwd(BF, FAKE, 8, FAKE, FAKE, FAKE, 1, None, FAKE, 8, 9, 4, 8, None) == -1                 # pitch < W
    assert bwd(BF, FAKE, 8, FAKE, FAKE, FAKE, 1, None, FAKE + 1, 8, 8, 4, 8, None) == -3
    assert lib.mmsum_sequence_logprob(FAKE, FAKE, 0, 3, 8, 0, FAKE, None) == -1
    pairs = lib.mmsum_preference_pairs
    assert pairs(FAKE, FAKE, None, 0, 3, 8, 0.1, 0.0, 0, FAKE, FAKE, FAKE, FAKE, FAKE, None) == -1
    assert pairs(FAKE, FAKE, None, 2, 3, 8, 0.1, 1.5, 0, FAKE, FAKE, FAKE, FAKE, FAKE, None) == -1
    assert pairs(FAKE, FAKE, None, 2 ** 20, 2 ** 20, 8, 0.1, 0.0, 0, FAKE, FAKE, FAKE, FAKE, FAKE, None) == -1
    pref = lib.mmsum_preference_loss
    assert pref(BF, FAKE, 8, FAKE, None, 2, 3, 8, 0.1, 0.0, 0, FAKE, FAKE, FAKE, FAKE, 8, 8, None, None) == -4
    assert pref(BF, FAKE, 8, FAKE, None, 2, 3, 8, 0.1, float("nan"), 0, FAKE, FAKE, FAKE, FAKE, 8, 8, FAKE, None) == -1
    assert lib.mmsum_preference_workspace(0, 3) == 0 and lib.mmsum_preference_workspace(2, 3) > 0
    pol = lib.mmsum_policy_loss
    assert pol(BF, FAKE, 8, FAKE, FAKE, None, FAKE, 0, 2, 3, 8, 0.2, 0.2, 0.0, 0, FAKE, FAKE, FAKE, 8, 8, None, None) == -4
    assert pol(BF, FAKE, 8, FAKE, FAKE, None, FAKE, 0, 2, 3, 8, -0.2, 0.2, 0.0, 0, FAKE, FAKE, FAKE, 8, 8, FAKE, None) == -1
    assert pol(9, FAKE, 8, FAKE, FAKE, None, FAKE, 0, 2, 3, 8, 0.2, 0.2, 0.0, 0, FAKE, FAKE, FAKE, 8, 8, FAKE, None) == -2
    assert lib.mmsum_policy_terms(FAKE, FAKE, FAKE, None, FAKE, 0, 2, 0, 8, 0.2, 0.2, 0.0, 0, FAKE, FAKE, FAKE, None) == -1
    assert lib.mmsum_embed_fwd(BF, FAKE, FAKE, 7, FAKE, 8, 4, 10, 8, 1.0, None) == -1 and lib.mmsum_embed_fwd(3, FAKE, FAKE, 8, FAKE, 8, 4, 10, 8, 1.0, None) == -2
    assert lib.mmsum_embed_fwd(0, FAKE, FAKE + 2, 8, FAKE, 8, 4, 10, 8, 1.0, None) == -3
    eb = lib.mmsum_embed_bwd
    assert eb(BF, FAKE, 8, FAKE, 4000, 10, 8, 1.0, -1, 0, FAKE, None, None) == -4 and eb(BF, FAKE, 8, FAKE, 2 ** 30, 10, 8, 1.0, -1, 0, FAKE, FAKE, None) == -1
    assert eb(BF, FAKE, 8, FAKE, 4, 10, 8, 1.0, -1, 0, FAKE, FAKE + 8, None) == -3 and eb(BF, FAKE, 7, FAKE, 4, 10, 8, 1.0, -1, 0, FAKE, FAKE, None) == -1
    assert lib.mmsum_quantize_i8(BF, FAKE, 8, 4, 8, FAKE, 65, FAKE, None) == -1 and lib.mmsum_quantize_i8(BF, FAKE, 8, 4, 8, FAKE + 8, 128, FAKE, None) == -3
    g8 = lib.mmsum_gemm_i8
    assert g8(FAKE, 128, FAKE, FAKE, 128, FAKE, None, BF, FAKE, 16, 4, 16, 100, 0, None) == -1
    assert g8(FAKE, 131200, FAKE, FAKE, 131200, FAKE, None, BF, FAKE, 16, 4, 16, 131200, 0, None) == -1
    assert g8(FAKE, 128, FAKE, FAKE, 128, FAKE, None, 5, FAKE, 16, 4, 16, 128, 0, None) == -2 and g8(FAKE + 4, 128, FAKE, FAKE, 128, FAKE, None, BF, FAKE, 16, 4, 16, 128, 0, None) == -3


def refused(exc, fn, *a, **k):
    with pytest.raises(exc):
        fn(*a, **k)


def test_python_entries_refuse():
    import multimodalsum_amd as mm
    from multimodalsum_amd import kernels as kn
    x, lab = torch.zeros(4, 3, 8), torch.zeros(4, 3, dtype=torch.int64)
    z, adv = torch.zeros(4, 3), torch.zeros(4)
    refused(RuntimeError, mm.sequence_logprobs, x, lab)                                    # CPU tensors: no fallback
    refused(TypeError, mm.sequence_logprobs, x, lab.int())
    refused(ValueError, mm.sequence_logprobs, x, lab[:, :2])
    refused(ValueError, mm.sequence_logprobs, x[0], lab[0])
    refused(ValueError, mm.sequence_logprobs, x[:0], lab[:0])
    refused(ValueError, mm.sequence_logprobs, x[:, :0], lab[:, :0])
    refused(ValueError, mm.sequence_logprobs, x.transpose(1, 2), torch.zeros(4, 8, dtype=torch.int64))
    refused(ValueError, mm.sequence_logprobs, x.expand(4, 3, 8)[:, ::2], lab[:, ::2])      # sequences further apart than their rows say
    refused(ValueError, mm.sequence_logprobs, x[:1].expand(4, 3, 8), lab)                  # the same rows twice
    refused(ValueError, mm.preference_loss_and_grad, x[:3], lab[:3])
    refused(ValueError, mm.preference_loss_and_grad, x, lab, torch.zeros(3))
    refused(TypeError, mm.preference_loss_and_grad, x, lab, torch.zeros(4, dtype=torch.float64))
    refused(ValueError, mm.preference_loss_and_grad, x, lab, label_smoothing=-0.1)
    refused(TypeError, mm.preference_loss_and_grad, x, lab, dlogits=x.bfloat16())
    refused(ValueError, mm.preference_loss_and_grad, x, lab, dlogits=torch.zeros(4, 3, 7))
    refused(ValueError, mm.preference_loss_and_grad, x.view(-1)[:64].view(2, 4, 8), torch.zeros(2, 4, dtype=torch.int64), dlogits=x.view(-1)[8:72].view(2, 4, 8))
    refused(TypeError, mm.preference_loss_and_grad, x.double(), lab)
    refused(ValueError, mm.PreferenceLoss(), x, lab, torch.zeros(4, requires_grad=True))
    refused(ValueError, mm.policy_loss_and_grad, x, lab, z, torch.zeros(3))
    refused(ValueError, mm.policy_loss_and_grad, x, lab, z[:, :2], adv)
    refused(ValueError, mm.policy_loss_and_grad, x, lab, z, adv, kl_coef=0.1)              # a KL term needs the reference
    refused(ValueError, mm.policy_loss_and_grad, x, lab, z, adv, clip_low=-0.1)
    refused(ValueError, mm.policy_loss_and_grad, x, lab, z, adv, reduction="sum")
    refused(ValueError, mm.ClippedPolicyLoss(), x, lab, z.clone().requires_grad_(True), adv)
    refused(RuntimeError, mm.policy_loss_and_grad, x, lab, z, adv)
    table = torch.zeros(10, 8)
    refused(RuntimeError, mm.scaled_embedding, lab, table)
    refused(TypeError, mm.scaled_embedding, lab.int(), table)
    refused(TypeError, mm.scaled_embedding, lab, table.half())
    refused(ValueError, mm.scaled_embedding, lab, table.t())
    refused(ValueError, mm.scaled_embedding_grad, torch.zeros(4, 2, 8), lab, 10)
    refused(ValueError, mm.scaled_embedding_grad, torch.zeros(4, 3, 8), lab, 10, accumulate=True)
    refused(ValueError, mm.scaled_embedding_grad, torch.zeros(4, 3, 8), lab, 10, out=torch.zeros(8, 10).t())
    refused(RuntimeError, mm.scaled_embedding_grad, torch.zeros(4, 3, 8), lab, 10)
    refused(RuntimeError, mm.Int8Linear, torch.zeros(4, 8))
    refused(ValueError, mm.Int8Linear, torch.zeros(4, 0))
    refused(ValueError, mm.Int8Linear, torch.zeros(4, 8), torch.zeros(3))
    refused(TypeError, mm.Int8Linear, torch.zeros(4, 8), out_dtype=torch.float16)
    refused(TypeError, kn.quantize_rows, torch.zeros(4, 8, dtype=torch.float16))
    refused(ValueError, kn.quantize_rows, torch.zeros(2, 131073))
    q, s = torch.zeros(4, 128, dtype=torch.int8), torch.zeros(4)
    refused(TypeError, kn.gemm_i8, q.int(), s, q, s, torch.zeros(4, 4))
    refused(ValueError, kn.gemm_i8, q[:, :64], s, q[:, :64], s, torch.zeros(4, 4))
    refused(ValueError, kn.gemm_i8, q, s, q, s, torch.zeros(4, 5))
    refused(TypeError, kn.gemm_i8, q, s, q, s, torch.zeros(4, 4, dtype=torch.float16))
    refused(ValueError, kn.gemm_i8, q, s[:3], q, s, torch.zeros(4, 4))
    refused(RuntimeError, kn.gemm_i8, q, s, q, s, torch.zeros(4, 4))
