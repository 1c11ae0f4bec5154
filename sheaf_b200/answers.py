"""Several answers to one prompt, with cached keys and values.

The sampling module (``Session.create_gpt_sampler``) restates
examples/nanogpt/sample.shf:28-45, whose window slides: every token's position
changes every step, so each step runs the whole window. While prompt and
answer fit the window nothing slides, positions stay what they were, and the
keys and values of earlier tokens can be kept. Here the prompt goes through
the model once, its keys and values are shared by all answers, and a step runs
one token of each answer:

    embedding -> per layer: layer norm, QKV product, append to the paged
    cache, attention to the shared prompt and the answer's own keys,
    projection; layer norm, MLP -> layer norm, head -> log probabilities

Parameters are the nanoGPT leaves in sorted-key order (as
``Session.create_gpt_vag`` takes them), in bf16 or f32.
"""
from __future__ import annotations

import numpy as np

from ._lib import ELEM_F32, ELEM_I32, lib
from .runtime import Buffer, Session, SheafB200Error


class Answers:
    """Draws answers to a prompt from a nanoGPT model.

    ``logits`` of the last step and ``scores`` stay on the device. The gradient
    of a policy-gradient step in them is ``Session.token_logprobs_vjp``; it ends
    at the logits, and nothing here takes it on to the parameters."""

    def __init__(self, session: Session, leaves: list[Buffer], *, n_layer: int, n_head: int, n_embd: int,
                 block_size: int, vocab_size: int, page_rows: int = 16):
        self.s, self.leaves = session, leaves
        self.n_layer, self.n_head, self.d = n_layer, n_head, n_embd
        self.block, self.v, self.page = block_size, vocab_size, page_rows
        self.elem = leaves[0].elem
        self.ld = -(-vocab_size // 8) * 8  # a logits row of whole 16-byte vectors
        self._adds: dict[int, str] = {}

    # -- products and sums -----------------------------------------------------
    def _matmul(self, a: Buffer, w: Buffer, c_elem: int, ld: int | None = None) -> Buffer:
        """a [m, k] @ w [n, k]^T -> [m, n], rows `ld` apart."""
        (m, k), n = a.shape, w.shape[0]
        ld = ld or n
        out = self.s.empty((m, ld), c_elem)
        size = lib().sb_op_matmul_workspace_size(self.elem, 0, 1, m, n, k)
        ws = self.s.empty((size // 4 + 1,), ELEM_F32)
        self._check("matmul", lib().sb_op_matmul(self.elem, a.device_ptr, k, 0, w.device_ptr, k, 1, m, n, k,
                                                 out.device_ptr, ld, c_elem, ws.device_ptr, size, self.s.stream))
        return out

    def _norm(self, x: Buffer, gamma: Buffer) -> Buffer:
        rows = x.shape[0]
        y = self.s.empty((rows, self.d), self.elem)
        mean, rstd = self.s.empty((rows,), ELEM_F32), self.s.empty((rows,), ELEM_F32)
        self._check("layernorm", lib().sb_op_layernorm_fwd(self.elem, x.device_ptr, gamma.device_ptr, y.device_ptr,
                                                           mean.device_ptr, rstd.device_ptr, rows, self.d,
                                                           self.s.stream))
        return y

    def _gelu(self, x: Buffer) -> Buffer:
        y = self.s.empty(x.shape, self.elem)
        self._check("gelu", lib().sb_op_gelu_fwd(self.elem, x.device_ptr, y.device_ptr, x.shape[0] * x.shape[1],
                                                 self.s.stream))
        return y

    def _add(self, a: Buffer, b: Buffer) -> Buffer:
        rows = a.shape[0]
        if rows not in self._adds:
            t = f"tensor<{rows}x{self.d}xf32>"
            self._adds[rows] = self.s.load_stablehlo(
                f"module @residual_{rows}_{self.d} {{\n  func.func @main(%arg0: {t}, %arg1: {t}) -> {t} {{\n"
                f"    %0 = stablehlo.add %arg0, %arg1 : {t}\n    return %0 : {t}\n  }}\n}}\n")
        return self.s.call(f"{self._adds[rows]}.main", [a, b])[0]

    @staticmethod
    def _check(what: str, rc: int) -> None:
        if rc:
            raise SheafB200Error(3, f"{what} failed ({rc})")

    def _ints(self, a) -> Buffer:
        return self.s.upload(np.asarray(a, np.int32), ELEM_I32)

    # -- the model ---------------------------------------------------------------
    def _forward(self, ids, first: int, each: int, append: dict, attend: dict) -> Buffer:
        """Logits [n, ld] (f32) of ids [n], `each` successive positions from `first` on a sequence."""
        n, d, P = len(ids), self.d, self.leaves
        ln_f, wpe, wte = P[1 + 6 * self.n_layer:]
        x = self.s.empty((n, d), ELEM_F32)
        row = d * (4 if self.elem == ELEM_F32 else 2)
        ids = self.s.upload(np.asarray(ids, np.float32), ELEM_F32)
        self._check("embedding", lib().sb_op_embedding_fwd(self.elem, ids.device_ptr, wte.device_ptr,
                                                           wpe.device_ptr + first * row, x.device_ptr, n, each, self.v,
                                                           d, self.s.stream))
        for i in range(self.n_layer):
            w_attn, w_proj, g1, g2, w_fc, w_fc2 = P[1 + 6 * i:7 + 6 * i]
            qkv = self._matmul(self._norm(x, g1), w_attn, self.elem)
            q = self.s.kv_append(self.caches[i], qkv, **append)
            o, _ = self.s.prefix_attention(self.caches[i], q, **attend)
            x = self._add(x, self._matmul(o, w_proj, ELEM_F32))
            u = self._matmul(self._norm(x, g2), w_fc, self.elem)
            x = self._add(x, self._matmul(self._gelu(u), w_fc2, ELEM_F32))
        return self._matmul(self._norm(x, ln_f), P[0], ELEM_F32, self.ld)

    def draw(self, prompt, n: int, n_new: int, *, k: int = 32, temperature: float = 1.0, seed: int = 0):
        """n answers of n_new tokens each to `prompt`, each token drawn from the k likeliest: tokens [n, n_new] (i32)
        and their log probabilities under the whole distribution at that temperature [n, n_new] (f32)."""
        prompt = np.asarray(prompt)
        T = len(prompt)
        if T < 1 or n < 1 or n_new < 1 or T + n_new - 1 > self.block:
            raise ValueError("prompt and answer have to fit the window")
        if k < 1:
            raise ValueError("a token has to be drawn from one alternative or more")
        k = min(k, self.v, 32)
        shared, own = -(-T // self.page), -(-n_new // self.page)
        self.caches = [self.s.kv_cache(shared + n * own, self.page, self.n_head, self.d // self.n_head, self.elem)
                       for _ in range(self.n_layer)]
        prompt_pages = self._ints(np.arange(shared)[None])
        pages = self._ints(shared + np.arange(n * own).reshape(n, own))
        # the prompt, once: one sequence that sees itself
        logits = self._forward(prompt, 0, T,
                               dict(seq=self._ints(np.zeros(T)), pos=self._ints(np.arange(T)), pages=prompt_pages),
                               dict(lens=self._ints([T]), pages=prompt_pages))
        rng = np.random.default_rng(seed)
        seq = self._ints(np.arange(n))
        tokens, logp = np.zeros((n, n_new), np.int32), np.zeros((n, n_new), np.float32)
        for step in range(n_new):
            self.logits = logits
            self.scores = self.s.token_logprobs(logits, self.v, temperature=temperature, k=k)
            ids, alt = (self.scores[name].to_host() for name in ("top_ids", "top_logp"))
            if step == 0:  # the prompt's last position is every answer's start
                ids, alt = np.repeat(ids[-1:], n, 0), np.repeat(alt[-1:], n, 0)
            p = np.exp(alt.astype(np.float64) - alt[:, :1])
            at = (rng.random((n, 1)) * p.sum(1, keepdims=True) >= p.cumsum(1)).sum(1).clip(max=k - 1)
            tokens[:, step], logp[:, step] = ids[np.arange(n), at], alt[np.arange(n), at]
            if step + 1 < n_new:
                logits = self._forward(tokens[:, step], T + step, 1,
                                       dict(seq=seq, pos=self._ints(np.full(n, T + step)), pages=pages, base=T),
                                       dict(lens=self._ints(np.full(n, step + 1)), pages=pages, prefix_pages=prompt_pages,
                                            prefix_len=T))
        self.s.check_device()
        return tokens, logp
