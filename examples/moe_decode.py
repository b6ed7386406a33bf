"""A feed-forward part with experts in 8-bit integers, as a decode loop and a prompt run it.

Random weights stand for a model's (no checkpoint is needed): what matters is the order of the calls. A layer is the
residual's addition and norm, the router's product, the choice of experts, their gate and up products, the products'
quantization, and the down products with the next residual. (A dense gate, up and down pair is the same calls with one expert: ids of
zeros [tokens, 1], weights of 1.) The decode step is captured into a graph once and replayed: every shape is the step's, and which experts
a token goes to stays on the device.

    python examples/moe_decode.py            # on a gfx950 GPU
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import densecore_amd as dc  # noqa: E402


class Experts:
    """The layer's weights in int8 with a scale per row, and the buffers of a step of up to `tokens` tokens."""

    def __init__(self, tokens, hidden=512, width=256, n_expert=32, top=4, seed=0, device="cuda"):
        self.hidden, self.width, self.n_expert, self.top = hidden, width, n_expert, top
        gen = torch.Generator(device=device)
        gen.manual_seed(seed)

        def weight(*shape):
            w = torch.randn((*shape[:-2], *shape[-2:]), generator=gen, device=device) / shape[-1] ** 0.5
            q, s = dc.quantize_i8(w.reshape(-1, shape[-1]))
            return q.view(shape), s.view(shape[:-1])
        self.norm = 1 + 0.1 * torch.randn(hidden, generator=gen, device=device)
        self.router, self.router_s = weight(n_expert, hidden)
        self.bias = 0.01 * torch.randn(n_expert, generator=gen, device=device)  # for balance: chooses, does not weigh
        self.gate, self.gate_s = weight(n_expert, width, hidden)
        self.up, self.up_s = weight(n_expert, width, hidden)
        self.down, self.down_s = weight(n_expert, hidden, width)
        empty = lambda *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device=device)  # noqa: E731
        slots = tokens * top
        self.q, self.s = empty(tokens, hidden, dtype=torch.int8), empty(tokens)
        self.logits = empty(tokens, n_expert)
        self.ids, self.weights = empty(tokens, top, dtype=torch.int32), empty(tokens, top)
        self.plan = empty(dc.moe_plan_size(tokens, top, n_expert), dtype=torch.uint8)
        self.h, self.hq, self.hs = empty(slots, width), empty(slots, width, dtype=torch.int8), empty(slots)
        need = [dc.moe_down_i8_workspace_size(tokens, top, hidden), dc.mul_mat_i8_workspace_size(tokens, n_expert, hidden), 256]
        self.workspace = empty(max(need), dtype=torch.uint8)

    def step(self, x, residual):
        """residual [tokens, hidden] fp32, in place: the layer before's output x is added, then this layer's."""
        dc.rms_norm_i8(x, self.norm, 1e-6, r=residual, h=residual, q=self.q, s=self.s)
        dc.mul_mat_i8(self.router, self.router_s, self.q, self.s, y=self.logits, workspace=self.workspace)
        dc.moe_route(self.logits, self.top, scoring="sigmoid", bias=self.bias, n_group=4, topk_group=2, group_best=2,
                     ids=self.ids, weights=self.weights)
        dc.moe_plan(self.ids, self.n_expert, plan=self.plan)
        dc.moe_gate_up_i8(self.plan, self.gate, self.gate_s, self.up, self.up_s, self.q, self.s, self.top, h=self.h)
        dc.quantize_i8(self.h, q=self.hq, s=self.hs)
        dc.moe_down_i8(self.plan, self.down, self.down_s, self.hq, self.hs, self.weights, r=residual, y=residual,
                       workspace=self.workspace)
        return residual


def reference(layer, x, residual):
    """The same layer in 64 bits, of the weights that the int8 rows stand for (the activations not quantized)."""
    f = lambda q, s: q.double() * s.double()[..., None]  # noqa: E731
    h = (x + residual).double()
    n = h / (h.square().mean(1, keepdim=True) + 1e-6).sqrt() * layer.norm.double()
    score = torch.sigmoid(n @ f(layer.router, layer.router_s).T)
    y = h.clone()
    for t in range(len(x)):
        ids = layer.ids[t].long()  # the choice is the layer's: borders may fall elsewhere
        w = score[t, ids] / score[t, ids].sum()
        for e, g in zip(ids.tolist(), w):
            gate, up = f(layer.gate[e], layer.gate_s[e]) @ n[t], f(layer.up[e], layer.up_s[e]) @ n[t]
            y[t] += g * (f(layer.down[e], layer.down_s[e]) @ (gate * torch.sigmoid(gate) * up))
    return y


def main(tokens=6, prompt=200, steps=4, device="cuda"):
    gen = torch.Generator(device=device)
    gen.manual_seed(1)
    layer, off = Experts(tokens, device=device), []
    x, r = (torch.randn((tokens, layer.hidden), generator=gen, device=device) for _ in range(2))
    out = torch.empty_like(r)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())  # which still makes the weights and inputs
    with torch.cuda.stream(stream):
        layer.step(x, out.copy_(r))  # once before the capture
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out.copy_(r)
        layer.step(x, out)
    for _ in range(steps):
        x.normal_(generator=gen)
        r.normal_(generator=gen)
        graph.replay()
        torch.cuda.synchronize()
        want = reference(layer, x, r)
        off.append(float((out - want).norm() / (want - x - r).norm()))
    # a prompt through the same weights, with buffers of its own
    big = Experts(prompt, device=device)
    x, r = (torch.randn((prompt, layer.hidden), generator=gen, device=device) for _ in range(2))
    got = big.step(x, r.clone())
    want = reference(big, x, r)
    off.append(float((got - want).norm() / (want - x - r).norm()))
    return off


if __name__ == "__main__":
    print("error of the layer's own part against 64 bits:", ", ".join(f"{v:.4f}" for v in main()))
