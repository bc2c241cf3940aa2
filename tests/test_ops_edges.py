"""The policy-head operators (factory_marl_amd/ops.py) at the edges of what they are defined for, on the CPU backend."""
import torch

from factory_marl_amd import ops

CPU = torch.device("cpu")


# ------------------------------------------------------------------ rows without a softmax
def softmaxless(device=CPU):
    """(logits, index, teacher): rows all barred, with +inf, with NaN, all barred with an empty list, ordinary"""
    inf, nan = float("inf"), float("nan")
    z = torch.randn(5, 9, generator=torch.Generator().manual_seed(1))
    z[0], z[1, 4], z[1, 2], z[2, 0], z[3] = -inf, inf, -inf, nan, -inf
    at = torch.tensor([[1, 5], [2, 5], [2, 5], [-1, -1], [2, 5]])
    return z.to(device), at.to(device), torch.tensor([[0.5, 1.0]] * 5).to(device)


def check_softmaxless(device):
    """a student whose row has no softmax has loss and gradient NaN, throughout; with nothing listed both are 0"""
    for dtype in (torch.float32, torch.bfloat16):
        for repeat in (1, 300):  # short and long rows
            z, at, t = softmaxless(device)
            leaf = z.repeat(1, repeat).to(dtype).requires_grad_()
            loss = ops.distill_loss(leaf, at, t)
            dz, = torch.autograd.grad(loss.sum(), leaf)
            assert loss[:3].isnan().all() and loss[3] == 0 and loss[4].isfinite()
            assert dz[:3].isnan().all() and not dz[3].any() and dz[4].isfinite().all()


def test_rows_of_the_student_without_a_softmax():
    check_softmaxless(CPU)
