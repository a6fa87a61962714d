"""The kernels that engines with 8-bit weights call, in 64-bit arithmetic on the CPU, beside `kernel_emulation.TorchKernels`."""

import torch

import plain_float8 as plain
from kernel_emulation import TorchKernels


class Float8Matrix:
    def __init__(self, whole, matrices):
        self.whole, self.matrices, self.shape, self.dtype, self.device = whole, matrices, whole.shape, torch.float8_e4m3fn, whole.device

    def dim(self):
        return 2


class Float8TorchKernels(TorchKernels):
    """Counts the products that go through 8-bit weights in `products`."""

    def __init__(self):
        super().__init__()
        self.products = 0

    def pack_float8(self, w, matrices=1):
        return Float8Matrix(plain.matrix(*plain.quantised_matrix(w.float(), matrices)), matrices)

    def gemm(self, a, w, out, accumulate=False, then_norm=None, full_sums=None):
        if not isinstance(w, Float8Matrix):
            return super().gemm(a, w, out, accumulate, **({} if then_norm is None else {"then_norm": then_norm}))
        assert full_sums is not None and then_norm is None
        self.products += 1
        y = plain.rows(a) @ w.whole.t()
        out.copy_((out.double() + y if accumulate else y).to(out.dtype))
        return None

    def gemm_swiglu(self, a, w, out, gate="silu"):
        if not isinstance(w, Float8Matrix):
            return super().gemm_swiglu(a, w, out, gate)
        assert w.matrices == 2
        self.products += 1
        y = plain.rows(a) @ w.whole.t()
        g, u = y[:, :out.shape[1]], y[:, out.shape[1]:]
        act = g * torch.sigmoid(g) if gate == "silu" else 0.5 * g * (1.0 + torch.tanh((2.0 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3)))
        out.copy_((act * u).to(out.dtype))

    def route_in_groups(self, logits, correction, chosen, weights, scoring="sigmoid", groups=1, keep=None, group_score="top2", renorm=True, factor=1.0,
                        experts=None):
        c, w = plain.route(logits[:, :experts], correction, chosen.shape[1], scoring, groups, groups if keep is None else keep, group_score, renorm, factor)
        chosen.copy_(c.to(torch.int32))
        weights.copy_(w.float())

    def experts_float8(self, x, chosen, weights, w_up, w_down, out, limit=float("inf"), alpha=1.0, shift=0.0, weigh_input=False, fresh=False, through=None,
                       full_sums=None):
        self.products += 2
        one = lambda w: (w.whole, torch.ones((w.matrices, -(-w.shape[0] // w.matrices // 128), -(-w.shape[1] // 128))))
        y, _ = plain.experts(x, chosen, weights, one(w_up), one(w_down), limit=limit, alpha=alpha, shift=shift, weigh_input=weigh_input, through=through)
        out.copy_((y if fresh else out.double() + y).to(out.dtype))
