"""A residual perceptron with layer norm, trained from 8-bit activation checkpoints and run in
8 bits:

    out = x + W2 act(W1 layer_norm(x) + b1) + b2.

Training computes in the parameters' type and keeps, of the three activations that the backward
pass needs, the 8-bit blocks: a value takes 1 byte and 1/128 of a scale instead of 4 or 2 bytes.
The weights' gradients are those of the restored values.  For inference the weights are quantised
once, in tiles of 128 x 128, and both products take 8-bit operands.

    python -m cudeep_amd.examples.perceptron8
"""
import torch

from .. import _lib as L
from .. import ops


def _product(a, b, transA=False, transB=False, bias=None):
    """op(a) op(b) (+ bias per column) in a's type."""
    kw = dict(transA=transA, transB=transB)
    if bias is not None:
        kw.update(bias=bias, bias_mode=L.BIAS_COL)
    if a.dtype == torch.float32:
        return ops.gemm(a, b, **kw)
    return ops.gemm16(a, b, **kw).to(a.dtype)


class Perceptron8:
    """Parameters as float32, float16 or bfloat16 tensors; biases b1 and b2 are float32."""

    def __init__(self, dim, hidden, *, act=L.EPI_GELU, dtype=torch.bfloat16, device="cuda", seed=0):
        g = torch.Generator().manual_seed(seed)

        def normal(rows, cols):
            return (torch.randn(rows, cols, generator=g) / cols ** 0.5).to(dtype).to(device)

        self.act = act
        self.gain = torch.ones(dim, dtype=dtype, device=device)
        self.shift = torch.zeros(dim, dtype=dtype, device=device)
        self.w1, self.w2 = normal(hidden, dim), normal(dim, hidden)
        self.b1 = torch.zeros(hidden, device=device)
        self.b2 = torch.zeros(dim, device=device)

    def parameters(self):
        return {"gain": self.gain, "shift": self.shift, "w1": self.w1, "b1": self.b1,
                "w2": self.w2, "b2": self.b2}

    def forward(self, x):
        """(out, what backward needs): x itself, its statistics and three Block8."""
        h, mean, rstd = ops.layer_norm(x, self.gain, self.shift, stats=True)
        h8 = ops.quantize8(h)
        z = _product(h, self.w1, transB=True, bias=self.b1)
        y, z8 = ops.activation8(z, self.act)
        y8 = ops.quantize8(y)
        out = x + _product(y, self.w2, transB=True, bias=self.b2)
        return out, (x, mean, rstd, h8, z8, y8)

    def backward(self, grad_out, kept):
        """(gradient of x, gradients by parameter name; those of weights and biases float32)."""
        x, mean, rstd, h8, z8, y8 = kept
        grads = {}
        grads["w2"], grads["b2"] = ops.linear_weight_grad8(grad_out, y8)
        dy = _product(grad_out, self.w2)
        dz = ops.activation_backward8(dy, z8, self.act)
        grads["w1"], grads["b1"] = ops.linear_weight_grad8(dz, h8)
        dh = _product(dz, self.w1)
        dx, grads["gain"], grads["shift"] = ops.layer_norm_backward(dh, x, mean, rstd, self.gain)
        return dx + grad_out, grads

    def quantised(self):
        """The weights for infer, laid out once."""
        return ops.quantize8(self.w1, tile_rows=128), ops.quantize8(self.w2, tile_rows=128)

    def infer(self, x, weights):
        w1, w2 = weights
        h = ops.layer_norm(x, self.gain, self.shift)
        y = ops.linear8(h, w1, self.b1, epilogue=self.act)
        return x + ops.linear8(y, w2, self.b2)


def train(model, x, target, steps, rate):
    """Gradient descent on the mean squared error; the losses."""
    losses = []
    for _ in range(steps):
        out, kept = model.forward(x)
        diff = out.float() - target.float()
        losses.append(float((diff * diff).mean()))
        _, grads = model.backward((diff * (2.0 / diff.numel())).to(x.dtype), kept)
        for name, p in model.parameters().items():
            p -= (rate * grads[name]).to(p.dtype)
    return losses


def main():
    torch.manual_seed(0)
    rows, dim, hidden = 2048, 256, 1024
    x = torch.randn(rows, dim, device="cuda")
    target = x + torch.sin(3.0 * x)
    model = Perceptron8(dim, hidden, dtype=torch.float32)
    losses = train(model, x, target, steps=200, rate=4.0)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {len(losses)} steps")
    _, kept = model.forward(x)
    small = sum(t.q.numel() + t.scale.numel() for t in kept[3:])
    whole = sum(t.q.numel() for t in kept[3:]) * x.element_size()
    print(f"checkpoints: {small} bytes, {whole} in the activations' type")
    full, _ = model.forward(x)
    out = model.infer(x, model.quantised())
    err = float((out - full).norm() / (full - x).norm())
    print(f"8-bit inference: {err:.4f} of the perceptron's output away from the full one")


if __name__ == "__main__":
    main()
