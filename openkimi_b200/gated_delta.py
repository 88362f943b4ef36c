"""The gated delta rule with one decay per head, next to KDA's decay per channel: chunkwise forward and backward, and its
recurrent forms for decoding.

    S~ = e^g S        e = beta (v - S~^T k)        S' = S~ + k e^T        o = scale S'^T q

q and k may have fewer heads than v (value head h goes with key head ``h // (HV // H)``), and K and V may differ.
"""

from __future__ import annotations

from functools import lru_cache

import torch

from . import _lib
from .ops import _cached_tables, _chunk_tables


def _flags(l2norm, gate, sigmoid, v_first):
    return ((_lib.FLAG_QK_L2NORM if l2norm else 0) | (_lib.FLAG_GATE if gate else 0) | (_lib.FLAG_BETA_SIGMOID if sigmoid else 0)
            | (_lib.FLAG_STATE_V_FIRST if v_first else 0))


@lru_cache(maxsize=64)
def _offsets(cu: tuple, device_index: int):
    return torch.tensor(cu, dtype=torch.int64, device=torch.device("cuda", device_index))


@torch.compiler.disable
def chunk_gated_delta_rule(q, k, v, g, beta, scale=None, initial_state=None, output_final_state=False,
                           use_qk_l2norm_in_kernel=False, use_gate_in_kernel=False, use_beta_sigmoid_in_kernel=False,
                           cu_seqlens=None, cu_seqlens_cpu=None, state_v_first=False, A_log=None, dt_bias=None):
    """Gated delta rule over whole sequences, differentiable in every floating argument.

    q, k: [B, T, H, K]; v: [B, T, HV, V]; g, beta: [B, T, HV] with HV a multiple of H and K, V in (64, 128); BF16 or FP32.  g is the
    natural-log decay of a token; with ``use_gate_in_kernel`` it is the gate's input and the decay ``-exp(A_log) * softplus(g +
    dt_bias)``, A_log and dt_bias [HV].  Decays below -1000 count as -1000.  ``use_qk_l2norm_in_kernel`` divides the rows of q and k by
    max(norm, 1e-6), ``use_beta_sigmoid_in_kernel`` takes beta as logits.  ``initial_state`` and the returned final state are FP32
    [N, HV, K, V], or [N, HV, V, K] with ``state_v_first``.

    ``cu_seqlens`` ([N+1], batch 1) packs N documents, each with a state of its own; ``cu_seqlens_cpu`` is the same on the host and
    saves a copy from the device (where both are given it is the one that counts).  Rows outside the documents have zero
    outputs and gradients.

    Sums, states and pairwise decays are in FP32; BF16 inputs are multiplied exactly and computed operands in 24 bits.  Of its norm a
    result in FP32 is about 4e-7 from 64 bits, and with BF16 inputs and K = V = 128 up to 6e-7 for states and 1.7e-6 for the gradients
    of g, beta, A_log and dt_bias.  At a decay below e^-104, 0 in FP32, the gradient of g is 0.  k and v are cast to the type of q, and
    g and beta to FP32 unless both are BF16.

    Differentiated calls keep about (4 K V + 256 V + 34000) bytes per 64 tokens and value head for the backward (BF16 with K = V =
    128: 173 KB).  Where long sequences are cut into segments (BF16, K = V = 128), every sequence and head has room for as many as the
    longest sequence, 8 K V bytes each in the forward and 4 K V in the backward: up to 1 GB and 0.5 GB.  The index tables of a call
    captured into a CUDA graph are kept for the life of the process.  A gradient is not differentiable again.  Returns
    ``(o [B, T, HV, V], final_state or None)``.
    """
    tables = (None, None, None, None, 0, 0, True)
    if cu_seqlens is not None or cu_seqlens_cpu is not None:
        host = cu_seqlens_cpu if cu_seqlens_cpu is not None else cu_seqlens.cpu()
        if host.dim() != 1 or host.numel() < 2:
            raise ValueError(f"cu_seqlens must be a vector of at least two offsets, got shape {tuple(host.shape)}")
        if q.dim() != 4:
            raise ValueError(f"q and k must have the same shape [B,T,H,K], got q={tuple(q.shape)}")
        if not q.is_cuda:
            raise RuntimeError("chunk_gated_delta_rule runs only on a CUDA device (sm_100a); there is no CPU fallback")
        if q.shape[0] != 1:
            raise ValueError(f"The batch size is expected to be 1 rather than {q.shape[0]} when using `cu_seqlens`.")
        tokens = q.shape[0] * q.shape[1]
        seq, off, nt, tab, longest = _chunk_tables(None, host, q.device, tokens)
        cu = tuple(int(x) for x in host.tolist())
        tables = (_cached_tables(_offsets, cu, q.device), seq, off, tab, nt, longest, cu[0] == 0 and cu[-1] == tokens)
    return _lib.host().chunk_gdr(q, k, v, g, beta, A_log, dt_bias, initial_state, scale,
                                 _flags(use_qk_l2norm_in_kernel, use_gate_in_kernel, use_beta_sigmoid_in_kernel, state_v_first),
                                 bool(output_final_state), *tables)


def recurrent_gated_delta_rule_step(q, k, v, g, beta, state, *, scale=None, A_log=None, dt_bias=None, use_qk_l2norm_in_kernel=False,
                                    use_gate_in_kernel=False, use_beta_sigmoid_in_kernel=False, state_v_first=False, inplace=False):
    """One decoding step of the gated delta rule.

    q, k: [N, H, K]; v: [N, HV, V]; g, beta: [N, HV]; ``state``: FP32 [N, HV, K, V] ([N, HV, V, K] with ``state_v_first``), e.g. the
    final state ``chunk_gated_delta_rule`` returned for the prompt; the switches mean what they mean there.  Returns
    ``(o [N, HV, V], new_state)``; with ``inplace=True`` the state tensor itself is updated and returned (an expanded one is
    refused).  Inference only (no autograd).
    """
    return _lib.host().recurrent_gdr(q, k, v, g, beta, state, A_log, dt_bias, scale,
                                     _flags(use_qk_l2norm_in_kernel, use_gate_in_kernel, use_beta_sigmoid_in_kernel, state_v_first),
                                     bool(inplace), False, True)


def fused_recurrent_gated_delta_rule(q, k, v, g, beta, scale=None, initial_state=None, output_final_state=False, *, A_log=None,
                                     dt_bias=None, use_qk_l2norm_in_kernel=False, use_gate_in_kernel=False,
                                     use_beta_sigmoid_in_kernel=False, state_v_first=False):
    """Token-by-token gated delta rule over ``[B, T, ...]`` inputs, the shapes and switches of ``chunk_gated_delta_rule`` (meant for the
    few tokens of a decode loop): the state stays on chip from the first token to the last.  Inference only.  Returns
    ``(o [B, T, HV, V], final_state or None)``."""
    return _lib.host().recurrent_gdr(q, k, v, g, beta, initial_state, A_log, dt_bias, scale,
                                     _flags(use_qk_l2norm_in_kernel, use_gate_in_kernel, use_beta_sigmoid_in_kernel, state_v_first),
                                     False, True, bool(output_final_state))
