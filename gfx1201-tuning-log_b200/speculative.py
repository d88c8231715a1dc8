"""Verification of drafted tokens against the target's probabilities
(csrc/spec_verify.cu through b200kv_spec_verify).

The target model is run on each sequence's last token and its drafts; row r's
logits say what follows token r, so row r verifies the token that was fed to row
r + 1.  Drafts are taken while uniforms[r] * q(d) < p(d); the first row that
does not take its draft emits a token of the residual max(p - q, 0), the last row
one of p, by the race argmax p(v) / noise(v).  The random numbers are the
caller's: uniforms ~ U[0, 1), noise ~ Exp(1) (torch.Tensor.exponential_).
"""
import torch

from _b200kv import check, lib


def verify(logits, tokens, cu_rows, uniforms, noise, temperature=None, draft_probs=None, out_tokens=None,
           num_accepted=None):
    """Returns (out_tokens int64 [rows], num_accepted int32 [seqs]).

    logits float32 or bfloat16 [rows, vocab] (rows may be strided); tokens int64
    [rows], the ids fed; cu_rows int32 [seqs + 1]; uniforms float32 [rows]; noise
    float32 [seqs, vocab], > 0; temperature float32 [seqs] (0: greedy; None: 1);
    draft_probs float32 [rows, vocab], row r the distribution its draft was drawn
    from (a sequence's last row is not read; None: drafts that were not drawn,
    such as tokens looked up in the prompt).  Rows cu_rows[s] .. of out_tokens
    hold the sequence's num_accepted[s] taken drafts, the emitted token, then -1.
    """
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("logits must be float32 or bfloat16")
    if tokens.dtype != torch.int64 or cu_rows.dtype != torch.int32:
        raise TypeError("tokens must be int64 and cu_rows int32")
    for name, t in (("uniforms", uniforms), ("noise", noise), ("temperature", temperature),
                    ("draft_probs", draft_probs)):
        if t is not None and t.dtype != torch.float32:
            raise TypeError(f"{name} must be float32")
    rows, vocab = logits.shape
    seqs = cu_rows.shape[0] - 1
    if tokens.shape != (rows,) or uniforms.shape != (rows,):
        raise ValueError(f"tokens and uniforms must be [{rows}]")
    if noise.shape != (seqs, vocab):
        raise ValueError(f"noise must be [{seqs}, {vocab}]")
    if temperature is not None and temperature.shape != (seqs,):
        raise ValueError(f"temperature must be [{seqs}]")
    if draft_probs is not None and draft_probs.shape != (rows, vocab):
        raise ValueError(f"draft_probs must be [{rows}, {vocab}]")
    if out_tokens is None:
        out_tokens = torch.empty_like(tokens)
    elif out_tokens.dtype != torch.int64 or out_tokens.shape != (rows,):
        raise TypeError(f"out_tokens must be int64 [{rows}]")
    if num_accepted is None:
        num_accepted = torch.empty(seqs, dtype=torch.int32, device=logits.device)
    elif num_accepted.dtype != torch.int32 or num_accepted.shape != (seqs,):
        raise TypeError(f"num_accepted must be int32 [{seqs}]")
    for name, t in (("tokens", tokens), ("cu_rows", cu_rows), ("uniforms", uniforms), ("temperature", temperature),
                    ("out_tokens", out_tokens), ("num_accepted", num_accepted)):
        if t is not None and not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    for name, t in (("logits", logits), ("noise", noise), ("draft_probs", draft_probs)):
        if t is not None and t.stride(1) != 1:
            raise ValueError(f"{name} must have unit innermost stride")
    check(lib.b200kv_spec_verify(
        logits.data_ptr(), logits.stride(0), 1 if logits.dtype == torch.bfloat16 else 0, tokens.data_ptr(),
        cu_rows.data_ptr(), uniforms.data_ptr(), noise.data_ptr(), noise.stride(0),
        temperature.data_ptr() if temperature is not None else None,
        draft_probs.data_ptr() if draft_probs is not None else None,
        draft_probs.stride(0) if draft_probs is not None else 0, out_tokens.data_ptr(), num_accepted.data_ptr(), seqs,
        rows, vocab, torch._C._cuda_getCurrentRawStream(logits.device.index)), "b200kv_spec_verify")
    return out_tokens, num_accepted
