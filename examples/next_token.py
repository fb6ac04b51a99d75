"""The end of a language model, trained and then used: residual update with its
norms, head, log probabilities.

    python examples/next_token.py

A small table is learned (each token has one that follows it).  Training runs
residual_norm, the head's product, token_logprob and the gradients of all
three; the head is then held in 4 bits and the chain is followed one token at
a time with residual_norm, quant4_matvec and token_logprob's alternatives.
"""
import ctypes
import os
import sys

import numpy as np

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "acedia-r_b200"))
import acediar as acd  # noqa: E402


def matmul(a, b):
    """a %*% b in float32, through the library's launcher (on the default stream)."""
    a, b = acd.contiguous(a), acd.contiguous(b)
    out = acd.empty_tensor((a.shape[0], b.shape[1]), "float")
    acd.lib().tensor_matmul_float32(*[ctypes.c_void_p(t.storage.data_ptr()) for t in (out, a, b)],
                                    *[ctypes.c_size_t(n) for n in (a.shape[0], b.shape[1], a.shape[1])])
    return out


class Model:
    """Tokens are columns: `stream` and `block` hold, for each token, the residual
    stream and the last block's output (fixed here), one column a token."""

    def __init__(self, vocabulary=500, width=256, seed=0):
        rng = np.random.default_rng(seed)
        new = lambda x: acd.as_tensor(x.astype(np.float32), dtype="float")  # noqa: E731
        self.vocabulary = vocabulary
        self.after = rng.permutation(vocabulary)  # the token that follows, from 0
        self.stream = new(rng.standard_normal((width, vocabulary)))
        self.block = new(rng.standard_normal((width, vocabulary)))
        self.w_pre = new(np.ones(width))
        self.w_post = new(np.ones(width))
        self.gate = new(np.full(width, 0.5))
        self.head = new(np.zeros((vocabulary, width)))
        self.head4 = None

    def step(self, rate):
        """One step of gradient descent on all tokens; the mean loss before it."""
        tokens = acd.as_tensor((self.after + 1).astype(np.int64), dtype="int64")
        n = self.vocabulary
        norm = acd.residual_norm(self.stream, self.block, self.w_pre, self.w_post, self.gate)
        logits = matmul(self.head, norm.y)
        lp = acd.token_logprob(logits, tokens)
        loss = -acd.tensor_to_scalar(acd.tensor_mean(lp.logprob))

        d_lp = acd.as_tensor(np.full(n, -1.0 / n, np.float32), dtype="float")
        d_logits = acd.token_logprob_grad(logits, tokens, lp.logsumexp, d_logprob=d_lp, inplace=True)
        d_head = matmul(d_logits, acd.transpose_view(norm.y))
        d_y = matmul(acd.transpose_view(self.head), d_logits)
        grad = acd.residual_norm_grad(None, d_y, norm.h, self.block, norm.rstd_h, norm.rstd_block, self.w_pre,
                                      self.w_post, self.gate)
        self.head = self.head - d_head * rate
        self.w_pre = self.w_pre - grad.d_w_pre * rate
        self.w_post = self.w_post - grad.d_w_post * rate
        self.gate = self.gate - grad.d_gate * rate
        return loss

    def quantise(self, group=64):
        """The head in 4 bits, one scale and zero point for each `group` inputs of a token."""
        self.head4, self.group = acd.quant4_encode(self.head, group=group, zeros=True), group

    def next(self, token, top=3):
        """The `top` likeliest tokens after `token` (from 0) and their log probabilities."""
        column = lambda t: acd.subset(t, None, token + 1)  # noqa: E731
        y = acd.residual_norm(column(self.stream), column(self.block), self.w_pre, self.w_post, self.gate).y
        logits = acd.quant4_matvec(self.head4.weights, self.head4.scales, y, group=self.group, zeros=self.head4.zeros)
        lp = acd.token_logprob(logits, None, top=top)
        return acd.as_array(lp.top_index) - 1, acd.as_array(lp.top_logprob)


def main(steps=25, rate=5.0, follow=8):
    model = Model()
    losses = [model.step(rate) for _ in range(steps)]
    print("loss %.4f -> %.4f over %d steps" % (losses[0], losses[-1], steps))
    model.quantise()
    token, right = 0, 0
    for _ in range(follow):
        index, logprob = model.next(token)
        right += int(index[0]) == model.after[token]
        print("after %3d: %s" % (token, ", ".join("%d (%.3f)" % (i, p) for i, p in zip(index, logprob))))
        token = int(index[0])
    print("%d of %d as the table has it" % (right, follow))
    return losses, right, follow


if __name__ == "__main__":
    main()
