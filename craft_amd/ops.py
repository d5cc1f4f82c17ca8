"""Tensor-level wrappers over the C ABI: allocate outputs with torch, enqueue the HIP kernels.

Every function maps 1:1 to an entry point of ``include/craft_hip.h``; "tokens" = channels-last fp32
``[B, N, C]`` (possibly a column slice of a wider buffer: pass ``t[..., a:b]`` views, their row stride
is forwarded as ``ld``).  No compute happens in Python.
"""
from __future__ import annotations

import contextlib
import functools
import math
import os
import threading
from typing import Optional, Sequence

import torch

from . import hip
from .hip import ACT_NONE, ACT_RELU, ACT_TANH, PREC_F32, PROB_DTYPE, call, pick, round_up


def _ld(t: torch.Tensor) -> int:
    """Row stride (in elements) of a tokens view [..., n, c] whose channel stride is 1."""
    if t.stride(-1) != 1:
        raise hip.CraftHipError("tokens view must have unit channel stride")
    return t.stride(-2)


def _check_rows(t: torch.Tensor):
    # rows of a [B, N, C] view must be uniformly strided: stride(0) == N * stride(1)
    if t.dim() == 3 and t.shape[0] > 1 and t.stride(0) != t.shape[1] * t.stride(1):
        raise hip.CraftHipError("tokens view must be uniformly row-strided")


def tokens_from_nchw(x: torch.Tensor, c_off: int = 0, C: Optional[int] = None, act: int = ACT_NONE, ln: bool = False,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """NCHW [B, Ctot, H, W] channels [c_off, c_off+C) -> tokens [B, H*W, C] (+activation, +LayerNorm)."""
    B, Ctot, H, W = x.shape
    C = Ctot - c_off if C is None else C
    x = x.contiguous()
    if out is None:
        out = torch.empty(B, H * W, C, device=x.device, dtype=torch.float32)
    _check_rows(out)
    call("craft_tokens", x, 1, B, Ctot, c_off, C, H * W, 0, act, int(ln), out, _ld(out))
    return out


def tokens_from_nchw_wide(x: torch.Tensor) -> torch.Tensor:
    """NCHW -> tokens for any channel count (chunks of <= 256 channels written into column slices)."""
    B, C, H, W = x.shape
    ld = round_up(C, 4)
    out = torch.empty(B, H * W, ld, device=x.device, dtype=torch.float32)
    if ld != C:
        out[..., C:].zero_()
    for c0 in range(0, C, 256):
        c1 = min(C, c0 + 256)
        tokens_from_nchw(x, c_off=c0, C=c1 - c0, out=out[..., c0:c1])
    return out[..., :C]


def tokens_norm(t: torch.Tensor, act: int = ACT_NONE, ln: bool = True, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """tokens -> (activation) -> LayerNorm over C -> tokens."""
    B, N, C = t.shape
    _check_rows(t)
    if out is None:
        out = torch.empty(B, N, C, device=t.device, dtype=torch.float32)
    call("craft_tokens", t, 0, B, C, 0, C, N, _ld(t), act, int(ln), out, _ld(out))
    return out


def tokens_slice(t: torch.Tensor, c_off: int, C: int, act: int = ACT_NONE, ln: bool = False,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """tokens columns [c_off, c_off+C) -> (activation) -> (LayerNorm) -> tokens [B, N, C]."""
    B, N, Ctot = t.shape
    _check_rows(t)
    if out is None:
        out = torch.empty(B, N, C, device=t.device, dtype=torch.float32)
    _check_rows(out)
    call("craft_tokens", t, 0, B, Ctot, c_off, C, N, _ld(t), act, int(ln), out, _ld(out))
    return out


def tokens_to_nchw(t: torch.Tensor, H: int, W: int) -> torch.Tensor:
    B, N, C = t.shape
    _check_rows(t)
    out = torch.empty(B, C, H, W, device=t.device, dtype=torch.float32)
    call("craft_tokens_to_nchw", t, _ld(t), B, C, N, out)
    return out


def pack_linear_weight(w: torch.Tensor, prec: int) -> torch.Tensor:
    """[Cout, Cin] fp32 -> craft_pack_weights' MFMA fragment order with Cin padded to a multiple of 32 by zero columns: the weight
    operand craft_linear / craft_linear_t / craft_motion_encoder's convc1 take with CRAFT_W_PACKED / CRAFT_W1X1_PACKED (bf16 / fp16 /
    f16x3)."""
    cout, cin = w.shape
    Kp = round_up(cin, 32)
    m = w.detach().float()
    if Kp != cin:
        m = torch.cat([m, torch.zeros(cout, Kp - cin, device=w.device)], dim=1)
    m = m.contiguous()
    planes = 2 if prec == hip.PREC_F16X3 else 1
    out = torch.empty(planes * round_up(cout, 32) * Kp, device=w.device, dtype=torch.bfloat16 if prec == hip.PREC_BF16 else torch.float16)
    call("craft_pack_weights", m, cout, Kp, prec, out)
    return out


def linear_pack(owner, name: str, w: torch.Tensor, prec: int) -> Optional[torch.Tensor]:
    """The packed copy of the nn.Linear / 1x1-conv weight ``w`` (2-D view) for the ``proj`` role of ``prec``, cached on the module
    ``owner`` under ``name`` and rebuilt when the parameter is updated in place or replaced; None when the product runs in fp32, under
    autograd (a training step re-packs through its own registry) or with CRAFT_NO_LINEAR_PACK (A/B switch)."""
    pp = pick(prec, "proj")
    if pp == PREC_F32 or not w.is_cuda or torch.is_grad_enabled() and w.requires_grad or os.environ.get("CRAFT_NO_LINEAR_PACK"):
        return None
    cache = owner.__dict__.setdefault("_linear_packs", {})
    key = (pp, hip.weights_epoch(), w.data_ptr(), w._version, w.device, tuple(w.shape))
    e = cache.get(name)
    if e is None or e[0] != key:
        with torch.no_grad():
            e = cache[name] = (key, pack_linear_weight(w, pp))
        torch.cuda.current_stream().synchronize()       # (once per weight update; the copy may be consumed on other HIP streams)
    return e[1]


def linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], prec: int,
           out: Optional[torch.Tensor] = None, packed: Optional[torch.Tensor] = None) -> torch.Tensor:
    """nn.Linear on tokens: [B, N, Cin] x [Cout, Cin]^T (+bias) -> [B, N, Cout].  ``packed``: ``linear_pack`` of the same weight (the
    product then reads the weights in MFMA fragment order, k_gemm_rows_wf)."""
    B, N, Cin = x.shape
    _check_rows(x)
    Cout = w.shape[0]
    if out is None:
        out = torch.empty(B, N, Cout, device=x.device, dtype=torch.float32)
    _check_rows(out)
    if packed is not None:
        call("craft_linear", x, _ld(x), packed, bias, out, _ld(out), B * N, Cin, Cout, pick(prec, "proj") | hip.W_PACKED)
    else:
        call("craft_linear", x, _ld(x), w.contiguous(), bias, out, _ld(out), B * N, Cin, Cout, pick(prec, "proj"))
    return out


def linear_t(x: torch.Tensor, w: torch.Tensor, ldt: int, prec: int, out: Optional[torch.Tensor] = None,
             Dv: int = 0, acc_order: bool = False, packed: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Per-sample transposed projection: yT[b][o][n] (row stride ldt >= N, tail zero), stored in the
    element type of the pv role (the type attn_apply consumes).  With ``Dv`` (the per-mode value width) and a 16-bit
    pv type the result is in the MFMA fragment order craft_attn_apply requires (same shape / footprint);
    ``acc_order``: the key order ``flash_attention`` requires instead."""
    B, N, Cin = x.shape
    _check_rows(x)
    Cout = w.shape[0]
    pv = pick(prec, "pv")
    if out is None:
        # the tail columns N .. ldt-1 must read as zero; without a tail (N a multiple of 32: every BASELINE size) the kernel writes
        # every element and the 29 MB zero fill per aggregator call (12 per forward at 448x1024) is skipped
        alloc = torch.empty if ldt == N else torch.zeros
        out = alloc(B, Cout, ldt, device=x.device, dtype=PROB_DTYPE[pv])
    frag = Dv if (Dv and pv != PREC_F32) else 0
    if acc_order:
        if not frag:
            raise hip.CraftHipError("acc_order needs a 16-bit pv type and Dv")
        frag |= hip.FRAG_ACC_ORDER
    if packed is not None and frag:                     # (``packed``: linear_pack of the same weight; fragment-order results only)
        call("craft_linear_t", x, _ld(x), packed, out, ldt, B, N, Cin, Cout, pv, frag, pick(prec, "proj") | hip.W_PACKED)
    else:
        call("craft_linear_t", x, _ld(x), w.contiguous(), out, ldt, B, N, Cin, Cout, pv, frag, pick(prec, "proj"))
    return out


def score_max(q: torch.Tensor, k: torch.Tensor, H8: int, W8: int, M: int, scale: float, prec: int,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Device-side global max of the raw scaled scores as an ordered uint32 (setrans.py:520-529)."""
    B, N, C = q.shape
    if out is None:
        out = torch.zeros(32, device=q.device, dtype=torch.int32)
    call("craft_score_max", q, _ld(q), k, _ld(k), B, H8, W8, M, C // M, scale, out, pick(prec, "score"))
    return out


def decode_ord(o: torch.Tensor) -> float:
    """Host decode of the ordered-uint max (diagnostics / tests only; forces a sync)."""
    u = int(o[0].item()) & 0xFFFFFFFF
    import struct
    if u == 0:
        return float("nan")
    bits = (u & 0x7FFFFFFF) if (u & 0x80000000) else (~u & 0xFFFFFFFF)
    return struct.unpack("<f", struct.pack("<I", bits))[0]


class CorrPyramid:
    """Un-normalised correlation pyramid + lazy global-LayerNorm statistics.  ``tiled``: levels 0 / 1 are stored per query as 8 x 16 /
    4 x 8 tiles (CRAFT_PYR_TILED: the patch one workgroup of the fused build kernel writes -- whole 128-byte lines); ``dense(l)`` gives
    the row-major image of any level."""

    def __init__(self, B: int, H8: int, W8: int, levels: int, device, tiled: bool = False):
        self.B, self.H8, self.W8, self.levels = B, H8, W8, levels
        self.tiled = bool(tiled) and levels == 4 and min(H8, W8) >= 8
        N = H8 * W8
        self.lv, self.dims = [], []
        h, w = H8, W8
        for l in range(levels):
            self.dims.append((h, w))
            if self.tiled and l < 2:
                th, tw = (8, 16) if l == 0 else (4, 8)
                self.lv.append(torch.empty(B * N, -(-h // th) * -(-w // tw) * th * tw, device=device, dtype=torch.float32))
            else:
                self.lv.append(torch.empty(B * N, h, w, device=device, dtype=torch.float32))
            h, w = h // 2, w // 2
        self.sums = torch.zeros(B, 2, device=device, dtype=torch.float64)
        self.mu_rstd = torch.empty(B, 2, device=device, dtype=torch.float32)

    def nbytes(self) -> int:
        """Algorithmic bytes of the pyramid (the image sizes; a tiled level's padding is not counted)."""
        return sum(self.lv[l].shape[0] * h * w * 4 for l, (h, w) in enumerate(self.dims))

    def dense(self, l: int) -> torch.Tensor:
        """Level l as [B*N, h, w] row-major images (a copy for a tiled level: tests / debugging)."""
        h, w = self.dims[l]
        if not (self.tiled and l < 2):
            return self.lv[l]
        th, tw = (8, 16) if l == 0 else (4, 8)
        nty, ntx = -(-h // th), -(-w // tw)
        t = self.lv[l].view(-1, nty, ntx, th, tw).permute(0, 1, 3, 2, 4).reshape(-1, nty * th, ntx * tw)
        return t[:, :h, :w].contiguous()

    def batch_slice(self, b0: int, b1: int) -> "CorrPyramid":
        """View of samples [b0, b1) (no copy): the refinement loop of a batch slice can run on its own stream."""
        v = CorrPyramid.__new__(CorrPyramid)
        v.B, v.H8, v.W8, v.levels, v.tiled, v.dims = b1 - b0, self.H8, self.W8, self.levels, self.tiled, self.dims
        N = self.H8 * self.W8
        v.lv = [t[b0 * N:b1 * N] for t in self.lv]
        v.sums, v.mu_rstd = self.sums[b0:b1], self.mu_rstd[b0:b1]
        return v


def fused_pyramid(C: int, M: int, prec, levels: int, H8: int, W8: int) -> bool:
    """True when ``corr_build`` will run the fused build + pyramid kernel (craft_corr_build_pyramid) -- the caller may then allocate a
    tiled CorrPyramid (its stores fill whole 128-byte lines)."""
    return (pick(prec, "score") == hip.PREC_F16X3 and M == 4 and C == 256 and levels == 4 and min(H8, W8) >= 8
            and not os.environ.get("CRAFT_NO_FUSED_PYRAMID"))


def corr_build(q: torch.Tensor, k: torch.Tensor, H8: int, W8: int, M: int, scale: float, pos_tab: Optional[torch.Tensor],
               pos_w: float, w_aggr: float, clamp_ord: Optional[torch.Tensor], pyr: CorrPyramid, do_norm: bool,
               prec: int) -> CorrPyramid:
    B, N, C = q.shape
    R = 0 if pos_tab is None else (pos_tab.shape[0] - 1) // 2
    sp = pick(prec, "score")
    # f16x3, 4 modes of 64: scratch for the pre-split (hi / lo fp16) copies of Q and K
    ws = torch.empty(4 * B * N * C, device=q.device, dtype=torch.float16) if (sp == hip.PREC_F16X3 and M == 4 and C == 256) else None
    tab = None if pos_tab is None else pos_tab.contiguous()
    lv = pyr.lv + [None] * (4 - len(pyr.lv))
    if ws is not None and len(pyr.lv) == 4 and min(H8, W8) >= 8 and not os.environ.get("CRAFT_NO_FUSED_PYRAMID"):
        # pyramid written from the tile that produced level 0 (no re-read of the 604 MB level 0 at 768x1024)
        call("craft_corr_build_pyramid", q, _ld(q), k, _ld(k), B, H8, W8, M, C // M, scale, tab, R, pos_w, w_aggr, clamp_ord,
             lv[0], lv[1], lv[2], lv[3], pyr.sums, ws, sp | (hip.PYR_TILED if pyr.tiled else 0))
        call("craft_corr_finish", lv[0], None, None, None, pyr.sums, pyr.mu_rstd, B, H8, W8, int(do_norm))
        return pyr
    if pyr.tiled:
        raise hip.CraftHipError("a tiled CorrPyramid can only be filled by the fused build (f16x3 scores, 4 modes of 64, 4 levels, H8, W8 >= 8)")
    call("craft_corr_build", q, _ld(q), k, _ld(k), B, H8, W8, M, C // M, scale, tab, R, pos_w, w_aggr, clamp_ord, pyr.lv[0], pyr.sums, ws, sp)
    call("craft_corr_finish", lv[0], lv[1], lv[2], lv[3], pyr.sums, pyr.mu_rstd, B, H8, W8, int(do_norm))
    return pyr


def corr_lookup(pyr, coords: torch.Tensor, radius: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """coords tokens [B, N, 2] -> tokens [B, N, V*levels*(2r+1)^2].  ``pyr`` is one CorrPyramid or, for the two-way
    correlation of ``--f1`` (corr.py:164-171), a list of V of them: level l then holds [volume 0 | volume 1 | ...]."""
    pyrs = list(pyr) if isinstance(pyr, (list, tuple)) else [pyr]
    B, N, _ = coords.shape
    win2 = (2 * radius + 1) ** 2
    V = len(pyrs)
    nch = pyrs[0].levels * win2 * V
    if out is None:
        out = torch.empty(B, N, nch, device=coords.device, dtype=torch.float32)
    co = coords.contiguous()
    for v, pv in enumerate(pyrs):
        lv = pv.lv + [None] * (4 - len(pv.lv))
        call("craft_corr_lookup", lv[0], lv[1], lv[2], lv[3], pv.levels | (hip.PYR_TILED if getattr(pv, "tiled", False) else 0), pv.mu_rstd, co,
             B, pv.H8, pv.W8, radius, out, _ld(out), win2 * V, win2 * v)
    return out


def attn_probs(q: torch.Tensor, k: torch.Tensor, H8: int, W8: int, M: int, scale: float, pos_tab: Optional[torch.Tensor],
               pos_w: float, mask_radius: int, clamp_ord: Optional[torch.Tensor], prec: int,
               out: Optional[torch.Tensor] = None, defer: bool = False, relpos=None, tiled: Optional[bool] = None) -> torch.Tensor:
    """P [B, M, N, ldp] (ldp = N rounded up to 32; the tail columns are zero).  ``defer=True``: P is left un-normalised
    (exp(logit - rowmax)) and carries its row sums as ``P.craft_rowsum`` [B, M, N]; ``attn_apply`` divides by them.
    Only for P that goes straight to ``attn_apply`` -- anything handed to a caller is normalised.
    ``tiled`` (deferred one-launch path only; default on, ``CRAFT_P_ROWMAJOR=1`` turns it off): P is returned in 32-query x 64-key
    tiles (``hip.P_TILED``; shape [B, M, N rounded up to 32, N rounded up to 64], ``P.craft_tiled`` / ``P.craft_n`` set) -- opaque to
    everything but ``attn_apply`` / ``probs_slice`` / ``probs_rowmajor``.
    ``relpos = (Hs [B, M, N, 2*H8-1], Ws [B, M, N, 2*W8-1], weight)``: per-query relative-position scores (gma.RelPosEmb)."""
    B, N, C = q.shape
    ldp = round_up(N, 32)
    if pick(prec, "pv") not in PROB_DTYPE:
        raise hip.CraftHipError("inference stores the attention probabilities in the pv type: fp32, bf16 or fp16 (f16x3 is a "
                                "training-only pv mode)")
    given_out = out
    if out is None:
        out = torch.empty(B, M, N, ldp, device=q.device, dtype=PROB_DTYPE[pick(prec, "pv")])
    R = 0 if pos_tab is None else (pos_tab.shape[0] - 1) // 2
    pvp, sp = pick(prec, "pv"), pick(prec, "score")
    if (defer and relpos is None and C // M == 32 and sp in (hip.PREC_F16, hip.PREC_F16X3) and pvp in (hip.PREC_F16, hip.PREC_BF16)
            and N < 65536 and not os.environ.get("CRAFT_NO_FUSED_PROBS")):
        # one launch of independent waves (craft_attn_probs_fused): maxima + P' + row sums, keys pre-split in fragment order
        rowsum = torch.empty(B, M, N, device=q.device, dtype=torch.float32)
        ws = torch.empty(B * M * ((N + 127) // 128) * 16384, device=q.device, dtype=torch.uint8)
        if tiled is None:
            tiled = given_out is None and not os.environ.get("CRAFT_P_ROWMAJOR")
        if tiled:
            ldp = round_up(N, 64)
            if given_out is None:
                out = torch.empty(B, M, round_up(N, 32), ldp, device=q.device, dtype=PROB_DTYPE[pvp])
            elif tuple(out.shape) != (B, M, round_up(N, 32), ldp):
                raise hip.CraftHipError("tiled probabilities need an out of shape [B, M, round_up(N, 32), round_up(N, 64)]")
        call("craft_attn_probs_fused", q, _ld(q), k, _ld(k), B, H8, W8, M, C // M, scale,
             None if pos_tab is None else pos_tab.contiguous(), R, pos_w, mask_radius, clamp_ord, out, ldp, rowsum, ws,
             pvp | (hip.P_TILED if tiled else 0), sp)
        out.craft_rowsum = rowsum
        if tiled:
            out.craft_tiled, out.craft_n = True, N
        return out
    if tiled:
        raise hip.CraftHipError("tiled probabilities exist only on the deferred one-launch path (craft_attn_probs_fused)")
    # row sums | scratch: row maxima, per-key-chunk partial sums (CRAFT_ATTN_CHUNK_KEYS = 1024)
    rowsum = torch.empty(2 + (N + 1023) // 1024, B, M, N, device=q.device, dtype=torch.float32) if defer else None
    rph, rpw, rpwt = (None, None, 0.0) if relpos is None else (relpos[0].contiguous(), relpos[1].contiguous(), float(relpos[2]))
    if relpos is not None and (tuple(rph.shape) != (B, M, N, 2 * H8 - 1) or tuple(rpw.shape) != (B, M, N, 2 * W8 - 1)):
        raise hip.CraftHipError("relpos tables must be [B, M, N, 2*H8-1] and [B, M, N, 2*W8-1]")
    call("craft_attn_probs", q, _ld(q), k, _ld(k), B, H8, W8, M, C // M, scale,
         None if pos_tab is None else pos_tab.contiguous(), R, pos_w, mask_radius, clamp_ord, rph, rpw, rpwt, out, ldp, rowsum,
         pick(prec, "pv"), pick(prec, "score"))
    if defer:
        out.craft_rowsum = rowsum[0]
    return out


def flash_supported(N: int, W8: int, d: int, Dv: int, prec: int) -> bool:
    """Shapes / precisions craft_flash_attention implements (anything else: attn_probs + attn_apply)."""
    return (d == 64 and Dv == 256 and pick(prec, "pv") == hip.PREC_F16 and pick(prec, "score") in (hip.PREC_F16, hip.PREC_F16X3)
            and N < 65536 and W8 >= 2)


def flash_attention(q: torch.Tensor, k: torch.Tensor, vT: torch.Tensor, H8: int, W8: int, M: int, Dv: int, scale: float,
                    pos_tab: Optional[torch.Tensor], pos_w: float, mask_radius: int, clamp_ord: Optional[torch.Tensor], prec: int,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """O [B, M, N, Dv] = softmax(scores) @ V in one pass (the probabilities never reach memory).  ``vT`` from
    ``linear_t(..., Dv=Dv, acc_order=True)`` with ldt = N rounded up to 32."""
    B, N, C = q.shape
    d = C // M
    ldt = vT.shape[-1]
    sp = pick(prec, "score")
    planes = 2 if sp == hip.PREC_F16X3 else 1
    ws = torch.empty(B * M * (8 * ((N + 255) // 256) + (N + 31) // 32) * (d // 16) * planes * 1024, device=q.device, dtype=torch.uint8)
    if out is None:
        out = torch.empty(B, M, N, Dv, device=q.device, dtype=torch.float32)
    R = 0 if pos_tab is None else (pos_tab.shape[0] - 1) // 2
    call("craft_flash_attention", q, _ld(q), k, _ld(k), vT, ldt, B, H8, W8, M, d, Dv, scale,
         None if pos_tab is None else pos_tab.contiguous(), R, pos_w, mask_radius, clamp_ord, out, ws, sp, pick(prec, "pv"))
    return out


def vt_stride(P: torch.Tensor) -> int:
    """Row stride (key extent) of the V^T operand that ``attn_apply`` expects beside ``P``: P's own row stride for a row-major P, N
    rounded up to 32 for a tiled one (whose key extent is rounded to 64: include/craft_hip.h, craft_attn_apply)."""
    return round_up(P.craft_n, 32) if getattr(P, "craft_tiled", False) else P.shape[-1]


def probs_slice(P: torch.Tensor, b0: int, b1: int) -> torch.Tensor:
    """Batch slice of an ``attn_probs`` result that keeps the deferred row sums attached."""
    v = P[b0:b1]
    rs = getattr(P, "craft_rowsum", None)
    if rs is not None:
        v.craft_rowsum = rs[b0:b1]
    if getattr(P, "craft_tiled", False):
        v.craft_tiled, v.craft_n = True, P.craft_n
    return v


def probs_rowmajor(P: torch.Tensor) -> torch.Tensor:
    """Row-major [B, M, N, N] copy of an ``attn_probs`` result in either layout (tests / debugging; still un-normalised when
    the row sums are deferred)."""
    if not getattr(P, "craft_tiled", False):
        return P[..., :P.shape[2]]
    B, M, Nr, ldp = P.shape
    N = P.craft_n
    return P.view(B, M, Nr // 32, ldp // 64, 32, 64).permute(0, 1, 2, 4, 3, 5).reshape(B, M, Nr, ldp)[:, :, :N, :N]


def probs_tiled(P: torch.Tensor, fill: float = 0.0) -> torch.Tensor:
    """Tiled (``hip.P_TILED``) copy of a row-major P [B, M, N, >= N] (torch ops, not a kernel: tests and callers that build P
    themselves); the padding rows are filled with ``fill`` (the kernels never write them and the consumer must not depend on them)."""
    B, M, N = P.shape[:3]
    Nr, ldp = round_up(N, 32), round_up(N, 64)
    full = torch.full((B, M, Nr, ldp), fill, device=P.device, dtype=P.dtype)
    full[:, :, :N, :N] = P[..., :N]
    full[:, :, :N, N:] = 0
    out = full.view(B, M, Nr // 32, 32, ldp // 64, 64).permute(0, 1, 2, 4, 3, 5).contiguous().view(B, M, Nr, ldp)
    rs = getattr(P, "craft_rowsum", None)
    if rs is not None:
        out.craft_rowsum = rs
    out.craft_tiled, out.craft_n = True, N
    return out


def attn_apply(P: torch.Tensor, vT: torch.Tensor, Dv: int, prec: int, out: Optional[torch.Tensor] = None,
               rows32: int = 0) -> torch.Tensor:
    """O[b][m] = P[b][m] @ V_m with vT [B, M*Dv, ldp] (16-bit: fragment order, ``linear_t(..., Dv=Dv)``) -> O [B, M, N, Dv].
    ``rows32`` (0 = chosen from the grid size; 4..7: 32-row groups per block of the 4-wave 16-bit kernel; 8 / 10 / 12 / 14: the 8-wave kernel
    with rows32 / 2 groups per row half -- CRAFT_PV_ROWS)."""
    B, M, N, ldp = P.shape
    tiled = getattr(P, "craft_tiled", False)
    if tiled:
        N = P.craft_n
        if not P.is_contiguous():
            raise hip.CraftHipError("tiled probabilities must be contiguous")
    if out is None:
        out = torch.empty(B, M, N, Dv, device=P.device, dtype=torch.float32)
    pv = pick(prec, "pv")
    if PROB_DTYPE[pv] != P.dtype:
        raise hip.CraftHipError(f"attention probabilities are {P.dtype} but the pv precision expects {PROB_DTYPE[pv]}")
    if vT.dtype != P.dtype:
        raise hip.CraftHipError(f"V^T is {vT.dtype} but P is {P.dtype}")
    if vT.shape[-1] != vt_stride(P):
        raise hip.CraftHipError(f"V^T has key extent {vT.shape[-1]}, attn_apply expects {vt_stride(P)} beside this P (ops.vt_stride)")
    call("craft_attn_apply", P, ldp, getattr(P, "craft_rowsum", None), vT, B, N, M, Dv, out,
         pv | (rows32 << hip.PV_ROWS_SHIFT) | (hip.P_TILED if tiled else 0))
    return out


def mode_pool_ln(O: torch.Tensor, x: torch.Tensor, w_agg: torch.Tensor, skip_coeff: torch.Tensor,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    B, M, N, C = O.shape
    _check_rows(x)
    if out is None:
        out = torch.empty(B, N, C, device=O.device, dtype=torch.float32)
    _check_rows(out)
    call("craft_mode_pool_ln", O, x, _ld(x), w_agg.contiguous().view(-1), skip_coeff, B, N, M, C, out, _ld(out))
    return out


def gma_residual(mf: torch.Tensor, O: torch.Tensor, gamma: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    B, N, C = mf.shape
    if out is None:
        out = torch.empty(B, N, C, device=mf.device, dtype=torch.float32)
    call("craft_gma_residual", mf, _ld(mf), O, gamma, B, N, C, out, _ld(out))
    return out


def convex_upsample(mask: torch.Tensor, flow: torch.Tensor, H8: int, W8: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    B = mask.shape[0]
    up = torch.empty(B, 2, 8 * H8, 8 * W8, device=mask.device, dtype=torch.float32) if out is None else out
    call("craft_convex_upsample", mask, flow, B, H8, W8, up)
    return up


def coords_init(flow_init: Optional[torch.Tensor], B: int, H8: int, W8: int, device):
    N = H8 * W8
    if flow_init is not None:
        if not flow_init.is_cuda:
            raise ValueError("flow_init must be on the GPU")
        if tuple(flow_init.shape) == (1, 2, H8, W8) and B > 1:
            flow_init = flow_init.expand(B, -1, -1, -1)        # the reference's `coords1 + flow_init` broadcasts a batch of 1
        if tuple(flow_init.shape) != (B, 2, H8, W8):
            raise ValueError(f"flow_init must be [{B}, 2, {H8}, {W8}] (1/8 resolution), got {tuple(flow_init.shape)}")
    c0 = torch.empty(B, N, 2, device=device, dtype=torch.float32)
    c1 = torch.empty_like(c0)
    fl = torch.empty_like(c0)
    call("craft_coords_init", None if flow_init is None else flow_init.contiguous().float(), B, H8, W8, c0, c1, fl)
    return c0, c1, fl


def conv2d_tokens(x: torch.Tensor, hw, w_packed: torch.Tensor, bias: torch.Tensor, cout: int, KH: int, KW: int, act: int,
                  prec: int, packed: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """nn.Conv2d (stride 1, same padding) + bias (+ReLU) on tokens [B, N, Cin] -> [B, N, Cout]."""
    B, N, Cin = x.shape
    _check_rows(x)
    if out is None:
        out = torch.empty(B, N, cout, device=x.device, dtype=torch.float32)
    call("craft_conv2d_nhwc", x, _ld(x), Cin, w_packed, bias, cout, KH, KW, act, out, _ld(out), B, hw[0], hw[1],
         prec | (hip.W_PACKED if packed else 0))
    return out


# ---- weight packing (layout plumbing, cached by the modules) --------------------------------------
def pack_conv(w: torch.Tensor) -> torch.Tensor:
    """[Cout, Cin, KH, KW] -> [Cout, KH, KW, Cin] contiguous."""
    return w.detach().permute(0, 2, 3, 1).contiguous().float()


class WeightPackRegistry:
    """Every conv-weight operand a training step packs (``pack_conv_weights``), remembered so that the NEXT steps re-pack all of them in ONE
    launch right after the optimizer update (craft_pack_conv_weights_batch) instead of one launch per operand as the forward / backward
    reach them (71 at configs[3]).  Owned by a ``train.Trainer``: it is the active registry only inside that trainer's steps, its entries
    hold the weight tensors (views of the optimizer's flat buffer: addresses are stable), and ``repack()`` is called by the trainer after
    ``optimizer.step()``.  An operand asked for while the registry is not fresh (first step, after a checkpoint load: ``invalidate``) is
    packed on the spot, as before."""

    def __init__(self, storage_ptr: Optional[int] = None):
        self.storage_ptr = storage_ptr      # only operands of weights that live in THIS storage (the optimizer's flat buffer) are remembered:
                                            # a temporary (torch.cat of two weights, a folded BatchNorm) has a new address every step
        self.entries = {}           # key -> [out tensor, (w0, w1) kept alive, fill arguments]
        self.fresh = False          # the outputs hold the CURRENT weights
        self._tables = None         # (jobs device tensor, prefix device tensor, n, blocks) for the current entry set
        self._epoch = None

    def invalidate(self):
        self.fresh = False

    @staticmethod
    def _versions(w0, w1):
        return (w0._version, w1._version if w1 is not None else -1)

    def lookup(self, key):
        """The packed operand if it holds the CURRENT weights: packed after the last raw-pointer update (the optimizer's epoch) AND the
        source tensors untouched since (their autograd version counters: load_state_dict / load_checkpoint / any in-place edit between
        steps moves them)."""
        if self.fresh and self._epoch == hip.weights_epoch():
            e = self.entries.get(key)
            if e is not None and e[3] == self._versions(*e[1]):
                return e[0]
        return None

    def remember(self, key, out, w0, w1, fill_args):
        if key not in self.entries:
            self._tables = None
        self.entries[key] = [out, (w0, w1), fill_args, self._versions(w0, w1)]

    def prepare(self):
        """Build (and validate) the batched job table for the current entry set on the host + one upload; raises before anything of the
        step's update is enqueued (Trainer calls it in front of optimizer.step())."""
        if not self.entries or self._tables is not None:
            return
        import ctypes
        lib = hip.load()
        nbytes = int(lib.craft_pack_conv_job_bytes())
        n = len(self.entries)
        buf = (ctypes.c_ubyte * (nbytes * n))()
        first, blocks = [0], 0
        for i, (out, (w0, w1), fa, _) in enumerate(self.entries.values()):
            cout0, cout1, Cin, KH, KW, a0, a1, b0, b1, transposed, prec = fa
            nb = int(lib.craft_pack_conv_job_fill(ctypes.byref(buf, i * nbytes), ctypes.c_void_p(w0.data_ptr()), cout0,
                                                  ctypes.c_void_p(w1.data_ptr() if w1 is not None else 0), cout1, Cin, KH, KW, a0, a1, b0, b1,
                                                  transposed, prec, ctypes.c_void_p(out.data_ptr())))
            if nb < 0:
                raise hip.CraftHipError(f"craft_pack_conv_job_fill failed with code {-nb}")
            blocks += nb
            first.append(blocks)
        dev = next(iter(self.entries.values()))[0].device
        jobs = torch.frombuffer(bytearray(buf), dtype=torch.uint8).to(dev)
        pref = torch.tensor(first, dtype=torch.int32).to(dev)
        self._tables = (jobs, pref, n, blocks)

    def repack(self):
        """All remembered operands from the current weights, one launch (enqueued on the current stream)."""
        if not self.entries:
            return
        self.prepare()
        jobs, pref, n, blocks = self._tables
        call("craft_pack_conv_weights_batch", jobs, pref, n, blocks)
        for e in self.entries.values():
            e[3] = self._versions(*e[1])
        self.fresh, self._epoch = True, hip.weights_epoch()


class _ActivePacks(threading.local):
    """The registry of the trainer whose step is running ON THIS THREAD (train.Trainer.step), else None: a second trainer or a validation
    forward on another thread sees its own slot (the backward modes of autograd.py are thread-local for the same reason)."""
    reg = None

    def __getitem__(self, i):
        return self.reg

    def __setitem__(self, i, v):
        self.reg = v


ACTIVE_WEIGHT_PACKS = _ActivePacks()


def pack_conv_weights(w0: torch.Tensor, prec: int, w1: Optional[torch.Tensor] = None, sel=None, transposed: bool = False) -> torch.Tensor:
    """nn.Conv2d weights [Cout, Cin, KH, KW] (w0 and optionally w1 concatenated along Cout) -> the MFMA fragment-order operand of the
    conv kernels in ONE launch (craft_pack_conv_weights): input channels ``sel`` = ((a0, a1), (b0, b1)) or None (all); ``transposed``:
    the operand of the input-gradient convolution (rows = selected input channels, taps flipped).  16-bit / f16x3 precisions."""
    w0 = w0.detach()
    w0 = w0 if w0.is_contiguous() else w0.contiguous()
    cout0, Cin, KH, KW = w0.shape
    cout1 = 0
    if w1 is not None:
        w1 = w1.detach()
        w1 = w1 if w1.is_contiguous() else w1.contiguous()
        cout1 = w1.shape[0]
        assert tuple(w1.shape[1:]) == (Cin, KH, KW)
    (a0, a1), (b0, b1) = sel if sel is not None else ((0, Cin), (0, 0))
    nsel, cout = (a1 - a0) + (b1 - b0), cout0 + cout1
    rows, Cp = (nsel, round_up(cout, 32)) if transposed else (cout, round_up(nsel, 32))
    planes = 2 if prec == hip.PREC_F16X3 else 1
    reg = ACTIVE_WEIGHT_PACKS[0]
    key = None
    if (reg is not None and w0.dtype == torch.float32 and (w1 is None or w1.dtype == torch.float32) and w0.is_cuda
            and (reg.storage_ptr is None or (w0.untyped_storage().data_ptr() == reg.storage_ptr
                                             and (w1 is None or w1.untyped_storage().data_ptr() == reg.storage_ptr)))):
        key = (w0.data_ptr(), w1.data_ptr() if w1 is not None else 0, cout0, cout1, Cin, KH, KW, a0, a1, b0, b1, bool(transposed), prec)
        hit = reg.lookup(key)
        if hit is not None:
            return hit                                       # packed by the trainer's batched launch after the last optimizer update
        e = reg.entries.get(key)
        out = e[0] if e is not None else None                # (same buffer every step: the batch job's output address is fixed)
    else:
        out = None
    if out is None:
        out = torch.empty(planes * round_up(rows, 32) * KH * KW * Cp, device=w0.device, dtype=torch.bfloat16 if prec == hip.PREC_BF16 else torch.float16)
    call("craft_pack_conv_weights", w0.float() if w0.dtype != torch.float32 else w0, cout0, w1, cout1, Cin, KH, KW, a0, a1, b0, b1, int(transposed), prec, out)
    if key is not None:
        reg.remember(key, out, w0, w1, (cout0, cout1, Cin, KH, KW, a0, a1, b0, b1, int(transposed), prec))
    return out


def pack_conv_prec(w: torch.Tensor, prec: int) -> torch.Tensor:
    """[Cout, Cin, KH, KW] -> the weight operand the KxK conv kernels take with W_PACKED (craft_pack_weights): fp32 stays
    [Cout, KH, KW, Cin]; bf16 / fp16 / f16x3 become MFMA fragment order [K/32][ceil(Cout/32)][planes][2][64][8] (flat)."""
    if prec != PREC_F32 and w.dtype == torch.float32:
        return pack_conv_weights(w, prec)
    wp = pack_conv(w)
    if prec == PREC_F32:
        return wp
    rows, K = wp.shape[0], wp[0].numel()
    planes = 2 if prec == hip.PREC_F16X3 else 1
    out = torch.empty(planes * round_up(rows, 32) * K, device=w.device, dtype=torch.bfloat16 if prec == hip.PREC_BF16 else torch.float16)
    call("craft_pack_weights", wp, rows, K, prec, out)
    return out


def pack_convf1(w: torch.Tensor) -> torch.Tensor:
    """[128, 2, 7, 7] -> [7*7*2, 128] (tap-major, output channel contiguous)."""
    return w.detach().permute(2, 3, 1, 0).reshape(-1, w.shape[0]).contiguous().float()


def pack_convf1_mfma(w: torch.Tensor, prec: int) -> torch.Tensor:
    """[128, 2, 7, 7] -> the matrix-core operand of convf1: rows = output channels, k = ky*16 + kx*2 + c (kx = 7 and k >= 112
    zero), K = 128, in craft_pack_weights' fragment order for ``prec`` (bf16 / fp16 / f16x3)."""
    co = w.shape[0]
    m = torch.zeros(co, 7, 8, 2, device=w.device, dtype=torch.float32)
    m[:, :, :7, :] = w.detach().float().permute(0, 2, 3, 1)
    m = torch.cat([m.reshape(co, 112), torch.zeros(co, 16, device=w.device)], dim=1).contiguous()
    planes = 2 if prec == hip.PREC_F16X3 else 1
    out = torch.empty(planes * round_up(co, 32) * 128, device=w.device, dtype=torch.bfloat16 if prec == hip.PREC_BF16 else torch.float16)
    call("craft_pack_weights", m, co, 128, prec, out)
    return out


# ------------------------------------------------------------------------------------------------
# LayerNorm with weights
# ------------------------------------------------------------------------------------------------
DTYPE_CODE = {torch.float32: PREC_F32, torch.bfloat16: hip.PREC_BF16, torch.float16: hip.PREC_F16}
LAYER_NORM_MAX_WIDTH = 16384


def _on_device(*tensors):
    """The tensors' common device (their own: kernels are enqueued on ITS current stream, whichever device is current)."""
    dev = tensors[0].device
    for t in tensors:
        if t is not None and t.device != dev:
            raise hip.CraftHipError(f"tensors on different devices: {dev} and {t.device}")
    if dev.type != "cuda":
        raise hip.CraftHipError("craft_amd HIP ops need device tensors (no CPU fallback)")
    return dev


def _on(dev):
    """A context in which ``dev`` is the current device."""
    return _NOTHING if dev.index == torch._C._cuda_getDevice() else torch.cuda.device(dev)


_NOTHING = contextlib.nullcontext()


def _norm_rows(x: torch.Tensor):
    """(x as rows of one stride, the stride): x itself where its leading axes are one run of rows, else a copy."""
    C = x.shape[-1]
    if x.is_contiguous():
        return x, C
    if x.dim() == 1:
        return x.contiguous(), C
    if x.stride(-1) == 1 or C == 1:
        lead = [(n, st) for n, st in zip(x.shape[:-1], x.stride()[:-1]) if n != 1]
        if not lead:
            return x, C
        if all(a[1] == b[0] * b[1] for a, b in zip(lead, lead[1:])):
            return x, lead[-1][1]
    return x.contiguous(), C


def _owns_its_elements(t: torch.Tensor) -> bool:
    """No two elements of t lie in one place."""
    extent = 1
    for st, n in sorted(zip(t.stride(), t.shape)):
        if n > 1:
            if st < extent:
                return False
            extent += (n - 1) * st
    return True


def _pieces(t: torch.Tensor):
    """(address, bytes that lie together, steps in bytes from one such piece to another, bytes from the first to behind the last)"""
    run, steps, extent, size = 1, [], 1, t.element_size()
    for st, n in sorted(zip(t.stride(), t.shape)):
        if n > 1 and st:
            extent += (n - 1) * st
            if st == run and not steps:
                run *= n
            else:
                steps.append(st * size)
    return t.data_ptr(), run * size, steps, extent * size


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """No element of a is one of b's: their ranges do not meet, or their pieces lie beside one another in every common step (slices of one projection)."""
    pa, ra, sa, ea = _pieces(a)
    pb, rb, sb, eb = _pieces(b)
    if pa + ea <= pb or pb + eb <= pa:
        return True
    step = math.gcd(*sa, *sb)
    return step > 0 and ra <= (pb - pa) % step <= step - rb


def _check_layer_norm(x, weight, bias, eps):
    dtype, shape = x.dtype, x.shape
    if dtype not in DTYPE_CODE:
        raise hip.CraftHipError(f"layer_norm: fp32, fp16 or bf16 rows, not {dtype}")
    if not shape or not 1 <= shape[-1] <= LAYER_NORM_MAX_WIDTH:
        raise hip.CraftHipError(f"layer_norm: a last axis of 1 .. {LAYER_NORM_MAX_WIDTH}, not {tuple(shape)}")
    if not eps >= 0:
        raise hip.CraftHipError("layer_norm: eps must not be negative")
    wt = None
    for t in (weight, bias):
        if t is None:
            continue
        if t.shape != shape[-1:] or (t.dtype != dtype and t.dtype != torch.float32):
            raise hip.CraftHipError(f"layer_norm: {'weight' if t is weight else 'bias'} must be [{shape[-1]}] of {dtype} or fp32, not {tuple(t.shape)} of {t.dtype}")
        if wt is not None and t.dtype != wt:
            raise hip.CraftHipError("layer_norm: weight and bias must have one type")
        wt = t.dtype
    _on_device(x, weight, bias)
    return wt or dtype


def _layer_norm(x, weight, bias, eps, out, stats: bool):
    """(out, mean, rstd): the rows' statistics with ``stats``, else None"""
    y, both = _layer_norm_fwd(x, weight, bias, eps, out, stats)
    return (y, *both) if stats else (y, None, None)


def _layer_norm_fwd(x, weight, bias, eps, out, keep: bool):
    """(out, the rows' means and reciprocal deviations [2, rows] or None)"""
    wt = _check_layer_norm(x, weight, bias, eps)
    C = x.shape[-1]
    rows = x.numel() // C
    given = out is not None
    if not given:
        out, ldy = x.new_empty(x.shape), C
    else:
        if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
            raise hip.CraftHipError("layer_norm: out must be of x's shape, type and device")
        y, ldy = _norm_rows(out)
        if y.data_ptr() != out.data_ptr() or (rows > 1 and ldy < C):
            raise hip.CraftHipError("layer_norm: out must be one run of rows with contiguous channels")
        ldy = ldy if rows > 1 else C
    # (a small call is as fast as its host: one tensor for both statistics, whose halves go by their addresses)
    stats = x.new_empty((2, rows), dtype=torch.float32) if keep else None
    if rows:
        xr, ldx = _norm_rows(x)
        if given and not (y.data_ptr() == xr.data_ptr() and (ldy == ldx or rows == 1)) and not _apart(y, xr):
            raise hip.CraftHipError("layer_norm: out may be x itself, and must not overlap it otherwise")
        mean = stats.data_ptr() if keep else None
        hip.call_on(x.device, "craft_layer_norm_fwd", xr, ldx, None if weight is None else weight.contiguous(), None if bias is None else bias.contiguous(),
                    rows, C, float(eps), DTYPE_CODE[x.dtype], DTYPE_CODE[wt], out, ldy, mean, mean + 4 * rows if keep else None)
    return out, stats


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """LayerNorm over the last axis (width up to 16384) of fp32 / fp16 / bf16 rows; weight and bias [C] of the rows' type or fp32, each optional.
    Statistics in fp32, the result rounded once to x's type.  ``out`` may be x, and must not overlap it otherwise.  ``tokens_norm`` is the weightless fp32 form
    of the model's tokens; the differentiable form is ``autograd.layer_norm``."""
    with torch.no_grad():
        return _layer_norm(x, weight, bias, eps, out, False)[0]


def layer_norm_bwd(x: torch.Tensor, weight: Optional[torch.Tensor], bias_type: Optional[torch.dtype], dy: torch.Tensor, mean: torch.Tensor,
                   rstd: torch.Tensor, need=(True, True, True)):
    """(dx, dweight, dbias) of ``layer_norm`` from its saved row statistics; ``need`` leaves gradients out."""
    wt = weight.dtype if weight is not None else bias_type or x.dtype
    rows = x.numel() // max(x.shape[-1], 1) if x.dim() else 0
    if dy.shape != x.shape or wt not in (x.dtype, torch.float32):
        raise hip.CraftHipError(f"layer_norm_bwd: dy {tuple(dy.shape)} of rows {tuple(x.shape)}, weights of {wt}")
    for t in (mean, rstd):
        if t.numel() != rows or t.dtype != torch.float32 or not t.is_contiguous():
            raise hip.CraftHipError(f"layer_norm_bwd: mean and rstd must be {rows} contiguous fp32 numbers")
    _check_layer_norm(x, weight, None, 0.0)
    _on_device(x, dy, mean, rstd)
    return _layer_norm_bwd(x, weight, wt, dy, mean.data_ptr(), rstd.data_ptr(), need)


def _layer_norm_bwd(x, weight, wt, dy, mean: int, rstd: int, need):
    C = x.shape[-1]
    rows = x.numel() // C
    dx, dw, db, ws = x.new_empty(x.shape) if need[0] else None, None, None, None
    # one block of 1024 threads for each compute unit (or fewer, where there are few rows): each leaves one partial sum of the weight's gradients
    blocks = min(rows, 256)
    if need[1] or need[2]:
        dw, db = x.new_empty((2, C), dtype=wt).unbind()
        ws = x.new_empty(blocks * 2 * C, dtype=torch.float32) if rows else None
        dw, db = dw if need[1] else None, db if need[2] else None
    if not rows:
        return dx, None if dw is None else dw.zero_(), None if db is None else db.zero_()
    xr, ldx = _norm_rows(x)
    g, ldg = _norm_rows(dy if dy.dtype == x.dtype else dy.to(x.dtype))
    hip.call_on(x.device, "craft_layer_norm_bwd", xr, ldx, g, ldg if rows > 1 else C, None if weight is None else weight.contiguous(), mean, rstd, rows, C,
                DTYPE_CODE[x.dtype], DTYPE_CODE[wt], dx, C, dw, db, ws, blocks)
    return dx, dw, db


# ------------------------------------------------------------------------------------------------
# orthogonalisation of updates
# ------------------------------------------------------------------------------------------------
NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)        # the quintic that takes (0, 1] near 1 in 5 steps
ORTHOGONALIZE_MAX_SIDE = 32768                   # the smaller side of a matrix
_ORTHOGONALIZE_SMALL = 256                       # smaller sides up to here take the kernels that live on latency: 60 matrices to a set of launches, else 16


@functools.lru_cache(maxsize=64)
def _newton_schulz_scales(coeffs):
    """Powers of two that bring the operands of the products just below fp16's largest number: a matrix' entries are bounded by its largest singular
    value, and those follow the polynomial from [0, 1]."""
    g = [i / 4096 for i in range(4097)]
    top = [1.0, 1.0, 1e-3]
    for a, b, c in coeffs:
        q = [b * x * x + c * x ** 4 for x in g]
        top = [max(top[0], *map(abs, g)), max(top[1], *(x * x for x in g)), max(top[2], *map(abs, q))]
        g = [a * x + y * x for x, y in zip(g, q)]
        if not max(map(abs, g)) <= 100.0:
            raise hip.CraftHipError(f"orthogonalize: coefficients {coeffs} let singular values grow without bound")
    return tuple(2.0 ** math.floor(math.log2(48000.0 / t)) for t in top)


def _newton_schulz_coeffs(steps, coeffs):
    flat = all(isinstance(c, (int, float)) for c in coeffs)
    rows = [tuple(float(x) for x in coeffs)] * steps if flat else [tuple(float(x) for x in c) for c in coeffs]
    if steps != len(rows) or not 1 <= steps <= 64 or any(len(r) != 3 or not all(math.isfinite(x) for x in r) for r in rows):
        raise hip.CraftHipError("orthogonalize: coeffs are three finite numbers, or three for each of 1 .. 64 steps")
    return tuple(rows)


def orthogonalize(mats: Sequence[torch.Tensor], steps: int = 5, coeffs=NEWTON_SCHULZ, eps: float = 1e-7, out: Optional[Sequence[torch.Tensor]] = None):
    """Every matrix of the list with its singular values moved towards 1: X = G / (|G|_F + eps), then ``steps`` times X <- a X + (b A + c A A) X with
    A = X X^T from the smaller side.  ``coeffs``: (a, b, c), or one triple a step.  fp32 / fp16 / bf16 matrices of any strides, the smaller side up to
    32768; fp32-class arithmetic whatever the type, one rounding at the end.  (Entries of X keep 2^-40 of |G|_F + eps: a matrix far below eps, whose result
    is about as small, loses its small entries; without an eps a matrix of zeros gives NaN.)  The whole list shares its launches.  ``out`` (may be ``mats``, and
    must not overlap another matrix of it): where the results go.  ``train.FlatMuon`` is the optimizer that uses it."""
    rows = _newton_schulz_coeffs(steps, coeffs)
    scales = _newton_schulz_scales(rows)
    if not 0 <= eps < float("inf"):
        raise hip.CraftHipError("orthogonalize: eps must be finite and not negative")
    mats = list(mats)
    if out is not None:
        out = list(out)
        if len(out) != len(mats):
            raise hip.CraftHipError("orthogonalize: out must be a list of the matrices' shapes, types and devices")
        # a long list is worked off in parts: a result must not lie where another matrix, or another result, does
        where = {}
        for i, o in enumerate(out):
            if o.numel() and where.setdefault(o.data_ptr(), i) != i:
                raise hip.CraftHipError("orthogonalize: two results in one place")
        if any(g.numel() and where.get(g.data_ptr(), i) != i for i, g in enumerate(mats)):
            raise hip.CraftHipError("orthogonalize: a result in the place of another matrix")
    res, groups, device = [], {}, None
    for i, g in enumerate(mats):                      # (a list of a model's matrices: a microsecond here is fifty)
        shape, code = g.shape, DTYPE_CODE.get(g.dtype)
        if len(shape) != 2 or code is None:
            raise hip.CraftHipError(f"orthogonalize: fp32, fp16 or bf16 matrices, not {list(shape)} of {g.dtype}")
        r, c = shape
        small, large = (r, c) if r < c else (c, r)
        if small > ORTHOGONALIZE_MAX_SIDE or large > 1 << 22:
            raise hip.CraftHipError(f"orthogonalize: {list(shape)}: the smaller side up to {ORTHOGONALIZE_MAX_SIDE}, the larger up to 2^22")
        if out is None:
            o, ldo = None, c
        else:
            o = out[i]
            if o.shape != shape or o.dtype != g.dtype or o.device != g.device:
                raise hip.CraftHipError("orthogonalize: out must be a list of the matrices' shapes, types and devices")
            ldo, so = o.stride()
            if so != 1 and c > 1 or ldo < c and r > 1:
                raise hip.CraftHipError("orthogonalize: out needs contiguous columns")
            ldo = max(ldo, c)
        if device is None:
            device = _on_device(g)
        elif g.device != device:
            _on_device(mats[0], g)
        if o is None:
            o = torch.empty(shape, device=device, dtype=g.dtype)
        res.append(o)
        if small:
            groups.setdefault((code, small > _ORTHOGONALIZE_SMALL), []).append((g, o, r, c, small, large, ldo))
    import ctypes
    if groups:
        flat = hip.carray(ctypes.c_float, [x for row in rows for x in row])
        with torch.no_grad(), _on(device):
            for (code, large), todo in groups.items():
                most, pad = (16, 128) if large else (60, 64)
                for i in range(0, len(todo), most):
                    jobs, keep, nbytes = [], [], 8192 + ((32 << 20) if large else 0)
                    for g, o, r, c, m, k, ldo in todo[i:i + most]:
                        ld, sc = g.stride()
                        if (sc != 1 and c > 1) or ld < 0:
                            g = g.contiguous()
                            ld = c
                            keep.append(g)
                        m, k = (m + pad - 1) // pad * pad, (k + pad - 1) // pad * pad
                        nbytes += 2048 + 12 * m * k + 8 * m * m
                        jobs += (g.data_ptr(), ld, o.data_ptr(), ldo, r, c)
                    ws = torch.empty(nbytes, device=device, dtype=torch.uint8)
                    call("craft_orthogonalize", hip.carray(ctypes.c_long, jobs), len(jobs) // 6, flat, steps, float(eps), *scales, code, ws, nbytes)
    return res


# ------------------------------------------------------------------------------------------------
# attention with a cap, a distance bias and causal / prefix / document masks
# ------------------------------------------------------------------------------------------------
def _in_place(t: torch.Tensor) -> bool:
    """The kernels can read t where it lies: contiguous head width, 16-byte steps from a 16-byte address, rows less than 16 MiB apart."""
    step = 16 // t.element_size()
    return (t.stride(3) == 1 and t.data_ptr() % 16 == 0 and all(n == 1 or (s >= 0 and s % step == 0) for n, s in zip(t.shape[:3], t.stride()))
            and (t.shape[1] == 1 or t.stride(1) * t.element_size() < 1 << 24))


def _strided(t: torch.Tensor) -> torch.Tensor:
    """t itself where the kernels can read it in place, else a copy (a contiguous tensor at an odd address too, which ``contiguous()`` would hand back)."""
    return t if _in_place(t) else t.clone(memory_format=torch.contiguous_format)


def _strides(t: torch.Tensor):
    return [0 if n == 1 else s for n, s in zip(t.shape[:3], t.stride())]


class AttentionPlan:
    """The checked arguments of one attention call."""

    def __init__(self, q, k, v, scale, cap, slopes, causal, prefix, docs, docs_k):
        err = hip.CraftHipError
        if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
            raise err("attention: q, k, v are [batch, tokens, heads, width]")
        if q.dtype not in DTYPE_CODE or k.dtype != q.dtype or v.dtype != q.dtype:
            raise err(f"attention: q, k, v of one type, fp32, fp16 or bf16, not {q.dtype}, {k.dtype}, {v.dtype}")
        B, Nq, H, D = q.shape
        Nk, Hk = k.shape[1:3]
        if k.shape != (B, Nk, Hk, D) or v.shape != k.shape:
            raise err(f"attention: shapes {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)} do not fit")
        if H < 1 or Hk < 1 or H % Hk:
            raise err(f"attention: {H} query heads are no multiple of {Hk} key heads")
        if D % 8 or not 8 <= D <= 128:
            raise err(f"attention: a head width that is a multiple of 8, up to 128, not {D}")
        if not 0 <= float(cap) <= 1e30:
            raise err("attention: cap must be positive, or 0 for none")
        if cap > 4096 and q.dtype != torch.float32:
            raise err("attention: a cap of 4096 at most in 16-bit types (scores would be off by cap 2^-22)")
        scale = D ** -0.5 if scale is None else float(scale)
        if not abs(scale) <= 1e30:
            raise err("attention: scale must be finite")
        if cap and not abs(scale) / cap <= 1e30:
            raise err("attention: scale / cap must not pass 1e30")
        if prefix is not None and not causal:
            raise err("attention: a prefix opens a causal mask: pass causal=True")
        if slopes is not None and (slopes.shape != (H,) or slopes.dtype != torch.float32):
            raise err(f"attention: slopes must be [{H}] of fp32")
        if slopes is not None and slopes.requires_grad and torch.is_grad_enabled():
            raise err("attention: slopes have no gradient here")
        if docs is None and docs_k is not None:
            raise err("attention: docs_k needs docs")
        if docs is not None and docs_k is None:
            if Nq != Nk:
                raise err("attention: docs alone serves q and k of one length; pass docs_k too")
            docs_k = docs
        for t, shape, name in ((prefix, (B,), "prefix"), (docs, (B, Nq), "docs"), (docs_k, (B, Nk), "docs_k")):
            if t is not None and (t.shape != shape or t.dtype != torch.int32):
                raise err(f"attention: {name} must be {list(shape)} of int32, not {list(t.shape)} of {t.dtype}")
        if max(B, Nq, Nk) >= 1 << 29:
            raise err("attention: sizes below 2^29")
        self.device = _on_device(q, k, v, slopes, prefix, docs, docs_k)
        self.dims = (B, Nq, Nk, H, Hk, D)
        self.q, self.k, self.v = _strided(q), _strided(k), _strided(v)
        self.scale, self.cap, self.causal = scale, float(cap), int(bool(causal))
        self.slopes, self.prefix, self.docs, self.docs_k = (None if t is None else t.contiguous() for t in (slopes, prefix, docs, docs_k))
        self.code = DTYPE_CODE[q.dtype]

    def range_bytes(self) -> int:
        B, Nq, Nk = self.dims[:3]
        return 0 if self.docs is None else 16 * B * ((Nq + 31) // 32 + (Nk + 31) // 32)

    def new(self, nbytes: int) -> Optional[torch.Tensor]:
        return torch.empty(nbytes, device=self.device, dtype=torch.uint8) if nbytes else None

    def shape(self, *more):
        import ctypes
        return hip.carray(ctypes.c_long, [*self.dims] + [s for t in (self.q, self.k, self.v, *more) for s in _strides(t)])

    def masks(self):
        return self.slopes, self.prefix, self.docs, self.docs_k

    def splits(self) -> int:
        """0: blocks of 128 queries.  Otherwise the kernel of few rows (the tokens times the query heads of a key head, 32 to a block), whose keys are split
        over so many blocks: two for each compute unit in all, a split at least 256 keys.

        Up to 64 rows always (16 bf16 tokens of 32 / 8 heads of 128 against 32768 keys: 47 us, blocks of 128 queries 688; against 512 keys 26 and 22, the join's
        launch).  More rows where the keys are long and their blocks few enough to be split in two: 64 such tokens 92 and 692 us, 256 of them 283 and 690.
        One split, 512 blocks, is about even (512 tokens 500 and 692, 32 of a batch of 16 1246 and 1126), 1024 blocks are not (1048 and 717).  Long is 2048 keys (1024: 26 and 22 us), for fp32, whose blocks take
        3.6 times as long for a key, 512 (26 and 43 us; 300 keys at width 64: 22 and 30).  Documents keep to the blocks, which pass over tiles of others."""
        B, Nq, Nk, H, Hk, D = self.dims
        rows = Nq * (H // Hk)
        blocks = B * Hk * ((rows + 31) // 32)
        if rows > 64 and (self.docs is not None or blocks > 256 or Nk < (512 if self.code == PREC_F32 else 2048)):
            return 0
        return max(1, min(512 // blocks, (Nk + 255) // 256))

    def forward(self, out: torch.Tensor, lse: Optional[torch.Tensor] = None, rest: Optional[torch.Tensor] = None):
        B, Nq, Nk, H, Hk, D = self.dims
        splits = 0 if lse is not None else self.splits()
        nbytes = self.range_bytes() if not splits else 4 * B * Nq * H * splits * (D + 2) if splits > 1 else 0
        with _on(self.device):
            call("craft_attention_fwd", self.q, self.k, self.v, self.shape(out), *self.masks(), self.scale, self.cap, self.causal, self.code, splits, out,
                 lse, rest, self.new(nbytes), nbytes)

    def saved(self):
        """(log-sums, the rest of the output's rounding or None) for the forward pass to fill and the backward pass to read."""
        B, Nq, Nk, H, Hk, D = self.dims
        if self.code == PREC_F32:
            return torch.empty(B, H, Nq, 2, device=self.device, dtype=torch.float32), None
        return torch.empty(B, H, Nq, device=self.device, dtype=torch.float32), torch.empty(B, Nq, H, D, device=self.device, dtype=self.q.dtype)

    def backward(self, out: torch.Tensor, lse: torch.Tensor, rest: Optional[torch.Tensor], go: torch.Tensor, need=(True, True, True)):
        """(dq, dk, dv); ``need`` leaves dq out, or dk and dv (one kernel makes both) where neither is wanted."""
        B, Nq, Nk, H, Hk, D = self.dims
        go = _strided(go.to(self.q.dtype))
        dq = torch.empty(B, Nq, H, D, device=self.device, dtype=self.q.dtype) if need[0] else None
        dk, dv = torch.empty(2, B, Nk, Hk, D, device=self.device, dtype=self.q.dtype) if need[1] or need[2] else (None, None)
        # key / value gradients of shared heads: one block walks over the group's heads, unless that leaves compute units without one of the two blocks they
        # hold.  (A block for each query head and a sum against it, us, causal, 2048 tokens, 4 key heads: 16 heads of 128 in bf16, 64 / 256 / 384 / 512 / 768 blocks:
        # 129 / 216 / 324 / 426 / 655 against 417 / 434 / 447 / 465 / 534; fp16 and fp32 of 64 cross at the same place; without a mask it lies at 384.)
        split_group = int(dk is not None and H > Hk and B * Hk * ((Nk + 127) // 128) < 512)
        up = lambda n: (n + 15) // 16 * 16                                 # noqa: E731
        nbytes = self.range_bytes() + up(4 * B * H * Nq) + split_group * 8 * B * Nk * H * D
        if self.code == hip.PREC_F16:                                      # (the largest norms, for the gradients' powers of two)
            each = 16 if D > 64 else 32
            nbytes += up(8 * B * Hk * min(1024, (max(Nq * (H // Hk), Nk) + each - 1) // each))
        with _on(self.device):
            call("craft_attention_bwd", self.q, self.k, self.v, out, rest, lse, go, self.shape(out, go), *self.masks(), self.scale, self.cap, self.causal, self.code,
                 split_group, dq, dk, dv, self.new(nbytes), nbytes)
        return dq, dk if need[1] else None, dv if need[2] else None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: Optional[float] = None, cap: float = 0.0, slopes: Optional[torch.Tensor] = None,
              causal: bool = False, prefix: Optional[torch.Tensor] = None, docs: Optional[torch.Tensor] = None, docs_k: Optional[torch.Tensor] = None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(z) v over the keys each query sees, z = cap tanh(scale q k / cap) - slope_h |pos_i - j|.

    q [B, Nq, H, D]; k, v [B, Nk, Hk, D] of the same type (fp32, fp16, bf16), H a multiple of Hk (query head h reads key head h // (H / Hk)), D a multiple
    of 8 up to 128; any strides (views the kernels cannot read in place are copied).  Query i stands at position i + Nk - Nq: new tokens at the end of a
    cache.  scale: 1 / sqrt(D) by default; cap 0: none; slopes [H] fp32.  ``causal``: keys up to the query's position, and with ``prefix`` [B] int32 also
    the first prefix[b] keys (a hidden key still counts as 0 times its v, which has to be finite).  ``docs`` [B, Nq] (and ``docs_k`` [B, Nk]) int32: only keys
    of the query's document; a negative document is padding, which nothing sees and whose rows of q, k, v may hold anything.  A query that sees nothing
    gives zeros.  Softmax sums and products accumulate in fp32; 16-bit types round the probabilities to their own type for the product with v, which leaves
    the result 1.2 to 1.4 times as far from the exact one as rounding it alone would.  ``flash_attention`` and ``attn_probs`` are the model's own forms over
    an image's tokens; the differentiable form is ``autograd.attention``.  ``out`` may be q, and must not overlap k or v."""
    with torch.no_grad():
        plan = AttentionPlan(q, k, v, scale, cap, slopes, causal, prefix, docs, docs_k)
        if out is None:
            out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not _in_place(out) or not _owns_its_elements(out):
            raise hip.CraftHipError("attention: out must be of q's shape, type and device, with 16-byte aligned rows of its own")
        elif out.numel():
            is_q = out.data_ptr() == plan.q.data_ptr() and _strides(out) == _strides(plan.q)
            for t, name in ((plan.q, "q"), (plan.k, "k"), (plan.v, "v")):
                if t.numel() and not (name == "q" and is_q) and not _apart(out, t):
                    raise hip.CraftHipError(f"attention: out must not share memory with {name}, which other blocks still read (it may be q itself)")
        if out.numel() and not k.shape[1]:
            return out.zero_()
        if out.numel():
            plan.forward(out)
        return out
