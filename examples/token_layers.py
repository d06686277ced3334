"""A small token model whose memory-bound parts run on thrust_b200: tokens are looked up, mixed along the sequence by a gated recurrence, sent to
experts and brought back, and scored against the same table; trained for a few steps, then used to write one token at a time.

    python examples/token_layers.py [--steps 30]

The matrix products are torch's; lookup, recurrence, dispatch and combination, and all their gradients, are the library's calls, wrapped as
torch.autograd functions below.  The text is made up: a walk on the tokens in which each is followed by one of two others, so that a
model which learns gets well below the loss of guessing, log(vocabulary).
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import thrust_b200 as tb  # noqa: E402


class Lookup(torch.autograd.Function):
    """rows = scale * table[tokens]; the gradient is the sum over each token's places."""

    @staticmethod
    def forward(ctx, table, tokens, scale):
        ctx.save_for_backward(tokens)
        ctx.rows, ctx.scale, ctx.dtype = table.shape[0], scale, table.dtype
        return tb.embedding(table, tokens, scale)

    @staticmethod
    def backward(ctx, grad):
        (tokens,) = ctx.saved_tensors
        return tb.embedding_grad(grad.contiguous(), tokens, ctx.rows, ctx.scale, dtype=ctx.dtype), None, None


class Recurrence(torch.autograd.Function):
    """h[t] = sigmoid(gate[t]) h[t-1] + (1 - sigmoid(gate[t])) x[t] along each of the packed sequences."""

    @staticmethod
    def forward(ctx, x, gate, offsets):
        h, last = tb.gated_scan(x, gate, None, offsets)
        ctx.save_for_backward(x, gate, h, offsets)
        ctx.mark_non_differentiable(last)
        return h, last

    @staticmethod
    def backward(ctx, grad, _):
        x, gate, h, offsets = ctx.saved_tensors
        dx, dgate, _ = tb.gated_scan_grad(grad.contiguous(), x, gate, h, None, None, offsets)
        return dx, dgate, None


class Dispatch(torch.autograd.Function):
    """Tokens' rows by expert, and the plan for the way back."""

    @staticmethod
    def forward(ctx, x, experts, num_experts):
        rows, plan = tb.expert_dispatch(x, experts, num_experts)
        ctx.plan = plan
        ctx.mark_non_differentiable(*plan)
        return (rows, *plan)

    @staticmethod
    def backward(ctx, grad, *_):
        return tb.expert_dispatch_grad(grad.contiguous(), ctx.plan), None, None


class Combine(torch.autograd.Function):
    """The experts' rows, weighted and added up for each token."""

    @staticmethod
    def forward(ctx, rows, weights, *plan):
        plan = tb.ExpertPlan(*plan)
        ctx.save_for_backward(rows, weights)
        ctx.plan = plan
        return tb.expert_combine(rows, plan, weights)

    @staticmethod
    def backward(ctx, grad):
        rows, weights = ctx.saved_tensors
        return (*tb.expert_combine_grad(grad.contiguous(), rows, ctx.plan, weights), None, None, None)


class TokenModel(torch.nn.Module):
    def __init__(self, vocabulary, dim, experts, choices):
        super().__init__()
        self.dim, self.experts, self.choices = dim, experts, choices
        make = lambda *shape: torch.nn.Parameter(torch.randn(*shape, device="cuda") / math.sqrt(shape[-2]))  # noqa: E731
        self.table = torch.nn.Parameter(0.05 * torch.randn(vocabulary, dim, device="cuda"))
        self.mix = make(dim, 2 * dim)                 # x and gate of the recurrence, in one product
        self.router = make(dim, experts)
        self.expert = make(experts, dim, dim)

    def route(self, h):
        weights, experts = torch.topk(h @ self.router, self.choices, dim=1)
        return torch.softmax(weights.float(), dim=1).contiguous(), experts

    def apply_experts(self, rows, offsets):
        ends = offsets.tolist()                       # how many rows each expert has: the host shapes the products by it
        parts = [rows[a:b] @ self.expert[e] for e, (a, b) in enumerate(zip(ends[:-1], ends[1:]))]
        return torch.nn.functional.silu(torch.cat(parts + [rows[ends[-1]:]]))

    def score(self, h):
        """Adds what the experts make of h, and scores every token of the table."""
        weights, experts = self.route(h)
        rows, *plan = Dispatch.apply(h, experts, self.experts)
        made = self.apply_experts(rows, plan[2])
        return (h + Combine.apply(made, weights, *plan)) @ self.table.t()

    def forward(self, tokens, offsets):
        x = Lookup.apply(self.table, tokens, math.sqrt(self.dim))
        both = x @ self.mix
        h, last = Recurrence.apply(both[:, :self.dim], both[:, self.dim:], offsets)      # halves of one tensor, as they lie
        return self.score(x + h), last

    @torch.no_grad()
    def step(self, tokens, state, slots):
        """One token of each sequence: state [pool, dim] is brought up to date, the next token's scores come back."""
        x = tb.embedding(self.table, tokens, math.sqrt(self.dim))
        both = x @ self.mix
        return self.score(x + tb.gated_step(both[:, :self.dim], both[:, self.dim:], state, slots))


def walks(generator, vocabulary, lengths):
    """Packed walks: token t is followed by 5 t + 1 or by 5 t + 2."""
    tokens = torch.randint(0, vocabulary, (len(lengths), max(lengths)), generator=generator)
    step = torch.randint(1, 3, tokens.shape, generator=generator)
    for t in range(1, tokens.shape[1]):
        tokens[:, t] = (5 * tokens[:, t - 1] + step[:, t]) % vocabulary
    offsets = torch.tensor([0] + list(lengths)).cumsum(0)
    return torch.cat([tokens[i, :n] for i, n in enumerate(lengths)]).cuda(), offsets.cuda()


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=30)
    args = ap.parse_args()
    vocabulary, lengths = 211, [700, 33, 1, 512, 250, 1000]
    torch.manual_seed(1)
    generator = torch.Generator().manual_seed(2)
    model = TokenModel(vocabulary, dim=128, experts=6, choices=2)
    optimizer = torch.optim.Adam(model.parameters(), lr=3e-3)
    losses = []
    for _ in range(args.steps):
        tokens, offsets = walks(generator, vocabulary, lengths)
        scores, _ = model(tokens, offsets)
        followed = torch.ones(tokens.numel(), dtype=torch.bool, device="cuda")
        followed[offsets[1:] - 1] = False             # the last token of a sequence is followed by nothing
        loss = torch.nn.functional.cross_entropy(scores[followed], tokens.roll(-1)[followed])
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    print("loss %.3f -> %.3f (guessing: %.3f)" % (losses[0], losses[-1], math.log(vocabulary)))
    # the scan over whole sequences and steps of one token give the same states
    with torch.no_grad():
        scores, last = model(tokens, offsets)
        state = torch.zeros(8, model.dim, device="cuda")
        slots = torch.tensor([5], device="cuda")
        first = tokens[offsets[1]:offsets[2]]
        for t in range(first.numel()):
            one = model.step(first[t:t + 1], state, slots)
    torch.testing.assert_close(state[5], last[1], rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(one[0], scores[offsets[2] - 1], rtol=1e-2, atol=1e-2)
    print("one token at a time: same states and scores")
    return losses


if __name__ == "__main__":
    main()
