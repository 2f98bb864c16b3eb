"""Training-step engine around the hot path (the loop body of the reference's engine.py:55-81):
flat parameter/gradient arenas, fused clip+AdamW, bucketed RCCL all-reduce overlapped with backward,
and an op-for-op PyTorch counterpart of the reference's matcher/loss (kept unchanged in behaviour).
"""
from __future__ import annotations

import inspect
import math
import os
import re
from typing import Dict, List, Optional, Sequence

import numpy as np
import torch
import torch.distributed as dist
from torch import nn

from . import ops

ALIGN = 64   # elements (256 B): every parameter starts on a 16-B-aligned, vector-friendly offset
# parameter-name prefixes of the hot path (pose_estimation_transformer.py:85-144 heads / input_proj; the transformer)
HOT_PREFIXES = ("input_proj.", "transformer.", "translation_head", "rotation_head", "query_embed.", "backbone.1.")
# ("backbone.1." = the Joiner's position embedding when it is a learned one (position_encoding.py:87-112): trained by the path's
# own backward (functional.PosEmbedFn).  It steps at the MAIN learning rate: the reference's lr_backbone group is
# lr_backbone_names = ['backbone.0'] (main.py:39,253-271), which matches the detector body only, never backbone.1.*)


_ENC_LAYER = re.compile(r"^transformer\.encoder\.layers\.(\d+)\.")


def _bucket_of(name: str, n_enc: int = 0) -> str:
    """Backward-completion order of the autograd nodes: heads -> decoder -> encoder layer n-1 ... 0 (one bucket each, the
    reference's DDP buckets, main.py:280-283) -> level_embed / the rest of the encoder -> input_proj.  Names sort in that order."""
    if name.startswith(("translation_head", "rotation_head")):
        return "0_heads"
    if name.startswith("transformer.decoder"):
        return "1_decoder"
    m = _ENC_LAYER.match(name)
    if m and n_enc:
        return f"2_encoder_{n_enc - 1 - int(m.group(1)):02d}"
    if name.startswith(("transformer.encoder", "transformer.level_embed")):
        return "2_encoder_99"
    return "3_input_proj"


class ParamArena:
    """All trainable parameters in ONE fp32 buffer (+ matching grad / Adam moment buffers).

    * kernels write parameter gradients straight into the grad arena (`p._grad_view`), so autograd
      never allocates, copies or accumulates a parameter gradient;
    * zero_grad is one memset, clip_grad_norm_ one reduction, AdamW one launch per LR group;
    * data parallel: buckets are contiguous arena ranges in backward-completion order, so each
      all-reduce is a single large RCCL call launched while the rest of backward still runs.
    Layout: parameters by bucket; the 0.1x learning rate of sampling_offsets (main.py:41) is a per-block multiplier table.
    Parameters that never receive a gradient in this configuration (transformer.reference_points.*
    in bbox mode; the reason the reference needs find_unused_parameters=True) stay outside, exactly as
    torch.optim.AdamW skips parameters whose .grad is None.
    muon: options of ops.MuonPlan.step / its `scale` as a dict (True or an empty one: the defaults; None or False: off) -- the weight matrices (MUON_SKIP: not the embeddings and tables, not the
    output layers: the heads' last ones and, in learned mode, the 2-row reference points) step by orthogonalised updates instead of AdamW, their first Adam moment being the momentum; learning rate,
    schedule, clip and weight decay are AdamW's (scale "rms" by default: steps of AdamW's size).  Self-attention's stacked in-projection
    counts as three matrices.  muon_blocks marks their blocks of 64 elements (poet_adamw_blocks leaves those alone).
    """
    MUON_SKIP = re.compile(r"level_embed|query_embed|^backbone\.|_head\w*\.\d+\.layers\.2\.|^transformer\.reference_points\.")

    def __init__(self, model: nn.Module, lr=2e-4, lr_proj_mult=0.1, proj_names=("reference_points", "sampling_offsets"),
                 weight_decay=1e-4, betas=(0.9, 0.999), eps=1e-8, exclude=("transformer.reference_points",), lr_backbone_mult=0.1, muon=None):
        muon = {} if muon is True else dict(muon) if muon or isinstance(muon, dict) else None
        self._check_muon(muon)
        if muon is not None and not lr >= 0:                  # (set_lr's factor, which the matrices take by its magnitude, would turn its sign)
            raise ValueError(f"ParamArena: with Muon updates the learning rate must not be negative, got {lr}")
        named = [(n, p) for n, p in model.named_parameters() if p.requires_grad and not any(e in n for e in exclude)]
        # Only the hot path's own parameters live here (their gradients are written by the HIP backward programs).  Anything
        # else that is trainable -- e.g. a real backbone, which the reference trains at lr_backbone (main.py:253-271) -- would
        # be weight-decayed every step without ever receiving a gradient: refuse it instead of mis-training it silently.
        stray = [n for n, _ in named if not n.startswith(HOT_PREFIXES)]
        if stray:
            raise ValueError(f"ParamArena: trainable parameters outside the hot path (freeze them or give them their own optimiser): {stray[:4]}"
                             f"{' ...' if len(stray) > 4 else ''}")
        is_proj = lambda n: any(k in n for k in proj_names)
        # Order: by bucket (backward-completion order), named_parameters order inside a bucket -- except that the two
        # query-side projections of every MSDeformAttn are laid out as [sampling_offsets.weight | attention_weights.weight]
        # and [sampling_offsets.bias | attention_weights.bias]: their outputs are the two column blocks of ONE activation
        # (offsets | logits), so with the parameters adjacent the pair is one (2+1)*M*L*P-wide Linear -- one GEMM forward,
        # one for dX, one for dW -- while state_dict still sees two nn.Linear modules.  The 0.1x learning rate of
        # sampling_offsets (main.py:41,253-271) is a per-64-element multiplier table instead of a separate arena range.
        byname = dict(named)
        n_enc = 1 + max([int(m.group(1)) for m in (_ENC_LAYER.match(n) for n, _ in named) if m] or [-1])
        bucket = lambda n: _bucket_of(n, n_enc)
        order, taken = [], set()
        # the value projections of ALL decoder layers read the same encoder memory: laid out adjacent (weights, then biases)
        # they are one (n_dec * d)-wide Linear -- one GEMM forward, one for dW, one for dX -- while state_dict still sees n_dec
        # separate modules (_link_value_stack)
        vw = sorted((n for n, _ in named if re.match(r"^transformer\.decoder\.layers\.\d+\.cross_attn\.value_proj\.weight$", n)),
                    key=lambda n: int(n.split(".")[3]))
        vb = [n[: -len("weight")] + "bias" for n in vw]
        vstack = vw + vb if len(vw) > 1 and all(b in byname for b in vb) else []
        for n, p in sorted(named, key=lambda t: bucket(t[0])):
            if n in taken:
                continue
            if vstack and n.startswith("transformer.decoder") and vstack[0] not in taken:
                for q in vstack:                              # first thing in the decoder bucket
                    order.append((q, byname[q]))
                    taken.add(q)
            if n.endswith("sampling_offsets.weight"):
                pre = n[: -len("sampling_offsets.weight")]
                quad = [pre + "sampling_offsets.weight", pre + "attention_weights.weight", pre + "sampling_offsets.bias", pre + "attention_weights.bias"]
                # encoder self-attention: the value projection's weight follows the pair -- d(src) = [d(offsets|logits) | d(value)
                # rows] [W_so ; W_aw ; W_v] is then ONE input-gradient product with K = 3 M L P + d (_link_projection_pairs: `_triple`)
                vname = pre + "value_proj.weight"
                if pre.startswith("transformer.encoder") and vname in byname and vname not in taken:
                    quad.insert(2, vname)
                if all(q in byname for q in quad):
                    for q in quad:
                        order.append((q, byname[q]))
                        taken.add(q)
                    continue
            order.append((n, p))
            taken.add(n)
        dev = named[0][1].device
        self.entries, off = [], 0
        self.buckets: List[tuple] = []
        cur, start = None, 0
        scale = []
        for n, p in order:
            b = bucket(n)
            if b != cur:
                if cur is not None:
                    self.buckets.append((cur, start, off))
                cur, start = b, off
            self.entries.append((n, p, off))
            size = -(-p.numel() // ALIGN) * ALIGN
            # lr_backbone applies to names matching 'backbone.0' only (main.py:39,253-271); HOT_PREFIXES keeps backbone.0.* out of the arena,
            # so this branch is for a caller that widens the prefixes -- backbone.1.* (learned position encoding) steps at the main lr
            scale += [lr_proj_mult if is_proj(n) else (lr_backbone_mult if "backbone.0" in n else 1.0)] * (size // ALIGN)
            off += size
        self.buckets.append((cur, start, off))
        self.n_main = off
        self.total = off
        self.flat = torch.zeros(off, dtype=torch.float32, device=dev)
        self.grad = torch.zeros(off, dtype=torch.float32, device=dev)
        self.m = torch.zeros(off, dtype=torch.float32, device=dev)
        self.v = torch.zeros(off, dtype=torch.float32, device=dev)
        self.sq = torch.zeros(1 + 1024, dtype=torch.float32, device=dev)       # [0] = sum of squares, [1:] = poet_sqnorm's partials
        # bf16 shadow of every weight: the second MFMA operand of the bf16 GEMMs; rewritten by the AdamW kernel
        self.flat_bf16 = torch.zeros(off, dtype=torch.bfloat16, device=dev)
        # ... and its bf16 residual (W = hi + lo to 16 mantissa bits): lets a split-weight product with a long K run as two
        # plain bf16 GEMMs, C = A hi^T then C += A lo^T (blocks.proj_ln_fwd)
        self.flat_bf16_lo = torch.zeros(off, dtype=torch.bfloat16, device=dev)
        for n, p, o in self.entries:
            k = p.numel()
            self.flat[o:o + k].copy_(p.data.reshape(-1))
            p.data = self.flat[o:o + k].view(p.shape)
            p._grad_view = self.grad[o:o + k].view(p.shape)
            p.grad = p._grad_view
            p._bf16 = self.flat_bf16[o:o + k].view(p.shape)
            p._bf16_lo = self.flat_bf16_lo[o:o + k].view(p.shape)
        self.refresh_shadow()
        # Learning rate = base_lr (a host scalar baked into captured graphs) x this per-64-element DEVICE table: the table
        # carries the 0.1x group of sampling_offsets AND the schedule (set_lr rescales it in place, so a replayed graph
        # follows a StepLR exactly like the eager path does; main.py:278 lr_scheduler.step()).
        self.muon_names = [n for n, p, _ in self.entries if p.dim() >= 2 and not self.MUON_SKIP.search(n)] if muon is not None else []
        self.muon_blocks = None
        if muon is not None:
            marks = [0] * len(scale)
            for n, p, o in self.entries:
                if n in set(self.muon_names):
                    for i in range(o // ALIGN, (o + p.numel() + ALIGN - 1) // ALIGN):
                        marks[i] = 1
            self.muon_blocks = torch.tensor(marks, dtype=torch.uint8, device=dev)
        self.lr_scale_base = torch.tensor(scale, dtype=torch.float32, device=dev)
        self.lr_scale = self.lr_scale_base.clone()
        self.base_lr = self.lr = float(lr)
        self.groups = [(0, self.total, lr)]
        self._link_projection_pairs()
        self._link_value_stack(vstack)
        self.weight_decay, self.betas, self.eps = weight_decay, betas, eps
        self.step_count = 0
        self.step_word = torch.zeros(1, dtype=torch.int32, device=dev)       # device copy of step_count (graph replays bump it)
        self.world = 1
        self.muon = None
        if muon is not None:
            self.muon = (self._muon_plan(muon.pop("scale", "rms")), muon)
        # model.load_state_dict copies into the fp32 arena views in place; the bf16 operand shadow must follow
        model.register_load_state_dict_post_hook(lambda module, incompatible: self.refresh_shadow())

    @staticmethod
    def _check_muon(opts):
        """Refuses options of the Muon step that its first call would refuse."""
        if opts is None:
            return
        known = ["scale"] + [k for k in inspect.signature(ops.MuonPlan.step).parameters if k != "self"]
        unknown = [k for k in opts if k not in known]
        if unknown:
            raise ValueError(f"ParamArena: unknown Muon options {unknown}, known are {known}")
        if opts.get("scale", "rms") not in ops.MUON_SCALES:
            raise ValueError(f"ParamArena: Muon's scale must be one of {sorted(ops.MUON_SCALES)}, got {opts['scale']!r}")
        ops._muon_options(**{k: v for k, v in opts.items() if k in ("momentum", "steps", "coeffs", "eps")})

    def _muon_plan(self, scale):
        if not self.flat.is_cuda:
            raise ValueError("ParamArena: Muon updates need the model on the GPU")
        mats = []
        for n, p, o in self.entries:
            if n in set(self.muon_names):
                parts = 3 if n.endswith("in_proj_weight") and p.shape[0] % 3 == 0 else 1
                r, c = p.shape[0] // parts, p.numel() // p.shape[0]
                mats += [(o + i * r * c, r, c, o // ALIGN) for i in range(parts)]
        view = lambda flat: [flat[o:o + r * c].view(r, c) for o, r, c, _ in mats]       # noqa: E731
        return ops.MuonPlan(view(self.flat), view(self.grad), view(self.m), scale=scale, p_bf16=view(self.flat_bf16), p_bf16_lo=view(self.flat_bf16_lo),
                            lr_scale=[self.lr_scale[b:b + 1] for _, _, _, b in mats])

    def set_lr(self, lr: float):
        """Scheduler entry (the reference's StepLR, main.py:277-278): effective from the next optimiser launch, eager or
        replayed.  The sampling_offsets group keeps its 0.1x ratio."""
        if self.muon is not None and not lr >= 0:             # (the matrices' learning-rate words count by their magnitude)
            raise ValueError(f"ParamArena.set_lr: with Muon updates the learning rate must not be negative, got {lr}")
        self.lr = float(lr)
        self.lr_scale.copy_(self.lr_scale_base * (self.lr / self.groups[0][2]))

    def step_lr(self, epoch: int, lr_drop: int, gamma: float = 0.1):
        """torch.optim.lr_scheduler.StepLR(optimizer, lr_drop) evaluated at `epoch` (main.py:277)."""
        self.set_lr(self.base_lr * gamma ** (epoch // lr_drop))

    def state_dict(self):
        """What the reference checkpoints as 'optimizer' + 'lr_scheduler' (main.py:293-301,364-372): Adam moments, step, lr."""
        if self.step_word.is_cuda:
            self.step_count = max(self.step_count, int(self.step_word.item()))
        sd = {"m": self.m.detach().cpu().clone(), "v": self.v.detach().cpu().clone(), "step": self.step_count,
              "lr": self.lr, "base_lr": self.base_lr, "names": [n for n, _, _ in self.entries]}
        if self.muon_names:
            sd["muon"] = list(self.muon_names)
        return sd

    def load_state_dict(self, sd):
        if list(sd["names"]) != [n for n, _, _ in self.entries]:
            raise ValueError("ParamArena.load_state_dict: parameter layout differs from the checkpoint's")
        if list(sd.get("muon", [])) != self.muon_names:
            raise ValueError("ParamArena.load_state_dict: the checkpoint's moments belong to another choice of optimiser (muon)")
        self.m.copy_(sd["m"]); self.v.copy_(sd["v"])
        self.step_count = int(sd["step"])
        self.step_word.fill_(self.step_count)
        self.base_lr = float(sd["base_lr"])
        self.set_lr(float(sd["lr"]))
        self.refresh_shadow()

    def _link_projection_pairs(self):
        """Hang the stacked views of every adjacent [sampling_offsets | attention_weights] pair on the sampling_offsets
        parameters (`_pair` = dict of fp32 / bf16 / gradient views of the (n_so + n_aw, d) weight and the bias)."""
        pos = {n: (p, o) for n, p, o in self.entries}
        for n, (w, o) in pos.items():
            if not n.endswith("sampling_offsets.weight"):
                continue
            pre = n[: -len("sampling_offsets.weight")]
            aw, sb, ab = (pos.get(pre + k) for k in ("attention_weights.weight", "sampling_offsets.bias", "attention_weights.bias"))
            if aw is None or sb is None or ab is None:
                continue
            (aw_p, aw_o), (sb_p, sb_o), (ab_p, ab_o) = aw, sb, ab
            if aw_o != o + w.numel() or ab_o != sb_o + sb_p.numel() or aw_p.shape[1] != w.shape[1]:
                continue                                     # not adjacent (odd sizes): the two Linears stay separate launches
            rows, d = w.shape[0] + aw_p.shape[0], w.shape[1]
            w._pair = dict(w=self.flat[o:o + rows * d].view(rows, d), w16=self.flat_bf16[o:o + rows * d].view(rows, d),
                           gw=self.grad[o:o + rows * d].view(rows, d), b=self.flat[sb_o:sb_o + rows], gb=self.grad[sb_o:sb_o + rows])
            vp = pos.get(pre + "value_proj.weight")
            if vp is not None and vp[1] == o + rows * d and vp[0].shape[1] == d:       # [W_so ; W_aw ; W_v]: bf16 operand of the merged dX
                r3 = rows + vp[0].shape[0]
                w._triple = dict(w16=self.flat_bf16[o:o + r3 * d].view(r3, d), w=self.flat[o:o + r3 * d].view(r3, d), n_oa=rows,
                                 gw=self.grad[o:o + r3 * d].view(r3, d))          # (the stacked GRADIENT: one weight-gradient launch for all three)

    def _link_value_stack(self, vstack):
        """Hang the stacked views of the decoder layers' value projections on layer 0's weight (`_vstack`: fp32 / bf16 /
        gradient views of the (n_dec * d, d) weight and the (n_dec * d) bias) when they really are contiguous."""
        if not vstack:
            return
        pos = {n: (p, o) for n, p, o in self.entries}
        n = len(vstack) // 2
        (w0, o0), (b0, ob) = pos[vstack[0]], pos[vstack[n]]
        d_out, d_in = w0.shape
        ok = all(pos[vstack[i]][1] == o0 + i * d_out * d_in and pos[vstack[i]][0].shape == w0.shape for i in range(n)) and \
            all(pos[vstack[n + i]][1] == ob + i * d_out for i in range(n))
        if not ok:
            return
        rows = n * d_out
        w0._vstack = dict(n=n, w=self.flat[o0:o0 + rows * d_in].view(rows, d_in), w16=self.flat_bf16[o0:o0 + rows * d_in].view(rows, d_in),
                          gw=self.grad[o0:o0 + rows * d_in].view(rows, d_in), b=self.flat[ob:ob + rows], gb=self.grad[ob:ob + rows])

    def refresh_shadow(self):
        """Re-derive the bf16 shadow from the fp32 masters (after construction / load_state_dict)."""
        if self.flat.is_cuda:
            ops.cast(self.flat, self.flat_bf16)
        else:
            self.flat_bf16.copy_(self.flat)
        self.flat_bf16_lo.copy_(self.flat - self.flat_bf16.float())

    def zero_grad(self):
        # (a CPU arena exists for the reducer's bookkeeping tests over gloo only -- no kernel ever runs on it)
        ops.zero_(self.grad) if self.grad.is_cuda else self.grad.zero_()

    def step(self, max_norm: float = 0.1, step_dev=None):
        """clip_grad_norm_(max_norm) + AdamW (engine.py:77-81) on the flat arenas.  With `step_dev` (a device word) the
        step count / bias corrections are read on the device, so the launch sequence can be replayed from a hipGraph."""
        gs = 1.0 / self.world
        sq = None
        if max_norm > 0:
            ops.zero_(self.sq) if self.sq.is_cuda else self.sq.zero_()
            ops.sqnorm(self.grad, self.sq)
            sq = self.sq
        if self.muon is not None:                             # (first: what it refuses, it refuses before anything has changed)
            plan, opts = self.muon
            plan.step(**{"lr": self.groups[0][2], "weight_decay": self.weight_decay, "sqnorm_buf": sq, "max_norm": max_norm, "grad_scale": gs, **opts})
        self.step_count += 1
        for a, b, lr in self.groups:
            if b > a:
                ops.adamw(self.flat[a:b], self.grad[a:b], self.m[a:b], self.v[a:b], b - a, lr, self.betas[0], self.betas[1],
                          self.eps, self.weight_decay, self.step_count, sqnorm_buf=sq, max_norm=max_norm, grad_scale=gs,
                          p_bf16=self.flat_bf16[a:b], step_dev=step_dev, lr_scale=self.lr_scale[a // ALIGN:],
                          p_bf16_lo=self.flat_bf16_lo[a:b], skip=None if self.muon_blocks is None else self.muon_blocks[a // ALIGN:])

    def grad_norm(self) -> torch.Tensor:
        return torch.sqrt(self.sq[0]) / self.world


# Stream capture in THREAD-LOCAL error mode: with a live RCCL process group its watchdog thread polls hipEventQuery on the
# work objects of earlier all-reduces, which the default (global) mode turns into hipErrorStreamCaptureUnsupported -- the
# watchdog then aborts the process in the middle of the capture.  Only this thread's calls need policing.
_CAPTURE = dict(capture_error_mode="thread_local")


def collectives_forced() -> bool:
    """POET_FORCE_COLLECTIVES=1: run the data-parallel machinery (broadcast, bucket all-reduces on the comm stream, segmented
    backward graphs) even in a 1-rank process group.  Lets a single-GPU box exercise the RCCL code path end to end."""
    return os.environ.get("POET_FORCE_COLLECTIVES", "0") not in ("", "0")


class BucketReducer:
    """Data-parallel gradient all-reduce (the reference's DDP, main.py:282): one process per GPU,
    `torch.distributed` backend 'nccl' == RCCL over xGMI.  Buckets are whole contiguous arena ranges;
    `bucket_done(tag)` is called from the end of each backward node, records an event on the compute
    stream and enqueues the all-reduce on a dedicated comm stream, so the collective of bucket k
    overlaps the backward of bucket k+1.  Sum-reduce here, the 1/world average is folded into the
    optimizer kernel (grad_scale).

    * The TAIL buckets (level_embed, input_proj: final only when backward is over) are never reduced on their own: `finish()`
      coalesces every adjacent un-reduced range into ONE collective, so exactly one small all-reduce (1.3 MB) is exposed at the
      end of backward -- the last encoder layer's bucket already runs under the input_proj backward.
    * grad_dtype=torch.bfloat16 (or POET_DP_GRAD_DTYPE=bf16): buckets travel as bf16 (24.5 MB instead of 49 MB per step over the
      153 GB/s xGMI links): cast into a staging buffer, all-reduce, cast back into the fp32 gradient arena, all on the comm
      stream; accumulation in the optimiser stays fp32.  Off by default: the sum over 8 ranks is then rounded to 8 mantissa bits
      per addition."""

    TAIL = ("2_encoder_99", "3_input_proj")

    def __init__(self, arena: ParamArena, group=None, grad_dtype=None):
        self.arena, self.group = arena, group
        self.world = dist.get_world_size(group) if dist.is_available() and dist.is_initialized() else 1
        self.active = self.world > 1 or (collectives_forced() and dist.is_available() and dist.is_initialized())
        arena.world = self.world
        self.on_gpu = arena.grad.is_cuda
        self.comm = torch.cuda.Stream() if (self.on_gpu and self.active) else None
        if grad_dtype is None:
            grad_dtype = torch.bfloat16 if os.environ.get("POET_DP_GRAD_DTYPE", "fp32").lower() in ("bf16", "bfloat16") else torch.float32
        if grad_dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("BucketReducer: grad_dtype must be float32 or bfloat16")
        self.grad_dtype = grad_dtype
        self.stage = None
        if self.active and grad_dtype == torch.bfloat16:
            self.stage = torch.empty(arena.total, dtype=torch.bfloat16, device=arena.grad.device)
        self.done = set()
        self.collectives = []                # (start, end) of every all-reduce of the current / last step

    def bucket_done(self, tag: str):
        if not self.active or tag in self.TAIL:
            return
        if not self.done:
            self.collectives = []
        for name, a, b in self.arena.buckets:
            if name == tag and name not in self.done:
                self.done.add(name)
                self._reduce(a, b)

    def _all_reduce(self, a, b):
        buf = self.arena.grad[a:b]
        if self.stage is None:
            dist.all_reduce(buf, op=dist.ReduceOp.SUM, group=self.group)
            return
        st = self.stage[a:b]
        if self.on_gpu:                      # HIP casts on the stream the collective runs on
            prev = ops._STREAM_OVERRIDE[0]
            ops._STREAM_OVERRIDE[0] = torch.cuda.current_stream().cuda_stream
            try:
                ops.cast(buf, st)
                dist.all_reduce(st, op=dist.ReduceOp.SUM, group=self.group)
                ops.cast(st, buf)
            finally:
                ops._STREAM_OVERRIDE[0] = prev
        else:                                # (CPU arenas exist in the gloo tests only)
            st.copy_(buf)
            dist.all_reduce(st, op=dist.ReduceOp.SUM, group=self.group)
            buf.copy_(st)

    def _reduce(self, a, b):
        self.collectives.append((a, b))
        if self.comm is not None:
            ev = torch.cuda.Event()
            ev.record(torch.cuda.current_stream())
            with torch.cuda.stream(self.comm):
                self.comm.wait_event(ev)
                self._all_reduce(a, b)
        else:
            self._all_reduce(a, b)

    def finish(self):
        """Reduce whatever was not reduced yet -- adjacent ranges as ONE collective --, then make the compute stream wait."""
        if not self.active:
            return
        if not self.done:
            self.collectives = []
        run = None
        for name, a, b in self.arena.buckets:
            if name in self.done:
                if run is not None:
                    self._reduce(*run)
                    run = None
                continue
            self.done.add(name)
            run = (a, b) if run is None else (run[0], b)
        if run is not None:
            self._reduce(*run)
        if self.comm is not None:
            torch.cuda.current_stream().wait_stream(self.comm)
        self.done.clear()


# ---- backward-completion hooks (set by the trainer; the autograd nodes call announce()) ----------------
_REDUCER: Optional[BucketReducer] = None


def set_reducer(r: Optional[BucketReducer]):
    global _REDUCER
    _REDUCER = r


def announce(tag: str):
    if _REDUCER is not None:
        _REDUCER.bucket_done(tag)


# ====================================================================================================
# matcher + loss: PyTorch counterpart of models/matcher.py:104-229 ('gt' mode) and
# models/pose_estimation_transformer.py:454-674 (translation + geodesic rotation losses)
# ====================================================================================================
class PoseMatcher(nn.Module):
    def __init__(self, cost_bbox: float = 1, cost_class: float = 1, bbox_mode: str = "gt", class_mode: str = "specific",
                 device_assign: bool = False):
        """device_assign ('gt' mode): SetCriterion runs the assignment ON THE GPU (poet_lsa_boxes: the algorithm SciPy's
        linear_sum_assignment uses, same tie-breaking) and gathers the matched targets there too -- no SciPy call, no
        host-built index arrays between the forward and backward graphs.  forward() below stays the host path."""
        super().__init__()
        if bbox_mode not in ("gt", "jitter", "backbone"):
            raise ValueError(f"PoseMatcher: unknown bbox_mode {bbox_mode!r}")
        self.cost_bbox, self.cost_class, self.bbox_mode, self.class_mode = cost_bbox, cost_class, bbox_mode, class_mode
        self.device_assign = bool(device_assign) and bbox_mode == "gt"
        self._cache = (None, None)

    @torch.no_grad()
    def forward(self, outputs, targets, n_boxes, giou_thresh=0.5):
        from scipy.optimize import linear_sum_assignment
        pb = outputs["pred_boxes"]
        if self.bbox_mode == "backbone":
            return self._forward_backbone(outputs, targets, n_boxes, giou_thresh)
        if self._cache[0] is pb:            # same boxes for every decoder layer: identical assignment
            return self._cache[1]
        bs, nq = pb.shape[:2]
        host = outputs.get("_pred_boxes_host")          # same values, already on the host: no device sync
        out_bbox = (np.asarray(host, dtype=np.float32) if host is not None else pb.detach().cpu().numpy()).reshape(bs, nq, -1)
        tgt_host = outputs.get("_tgt_boxes_host")        # host copy made by PoET.host_queries for this very batch
        if tgt_host is None:                             # standalone use: copy now (one transfer; blocks like matcher.py:139 does)
            from .modules import _to_host_list
            tgt_host = _to_host_list([t["boxes"] for t in targets], np.float32)
        if self.bbox_mode == "jitter":
            # matcher.py:175-181: the queries carry perturbed boxes, so the match is by class only (cost 0 = same class, 1 =
            # different); same cost matrix + same SciPy solver as the reference => the same tie-breaking
            pc, tl = outputs.get("_pred_classes_host"), outputs.get("_tgt_labels_host")
            if pc is None:
                pc = outputs["pred_classes"].detach().cpu().numpy()
            if tl is None:
                from .modules import _to_host_list
                tl = _to_host_list([t["labels"] for t in targets], np.int64)
            res = []
            for i in range(bs):
                c = self.cost_class * (np.asarray(pc[i][: n_boxes[i], None]) != np.asarray(tl[i])[None, :]).astype(np.float32)
                r, cidx = linear_sum_assignment(c)
                res.append((torch.as_tensor(r, dtype=torch.int64), torch.as_tensor(cidx, dtype=torch.int64)))
            self._cache = (pb, res)
            return res
        res = []
        for i, t in enumerate(targets):
            # L1 cost matrix of matcher.py:60-75 in numpy: the matrices are <= 20 x 20, and a torch CPU op here would wake
            # the whole OpenMP pool every step (its spinning workers eat the container's CPU quota and the process gets
            # descheduled for tens of ms while the GPU queue runs dry)
            tb = tgt_host[i]
            c = self.cost_bbox * np.abs(out_bbox[i, : n_boxes[i], None, :] - tb[None, :, :]).sum(-1)
            r, cidx = linear_sum_assignment(c)
            res.append((torch.as_tensor(r, dtype=torch.int64), torch.as_tensor(cidx, dtype=torch.int64)))
        self._cache = (pb, res)
        return res

    def _forward_backbone(self, outputs, targets, n_boxes, giou_thresh):
        """matcher.py:183-229, the mode pose_evaluate / bop_evaluate run (engine.py:127,212): the queries are detector boxes,
        so the cost is the L1 distance of the box CENTRES plus 0 / 1 for equal / different class, and a match survives only
        if the classes agree (class_mode 'specific') and the generalised IoU reaches `giou_thresh`.  Evaluation-side host
        code: float32 numpy in the reference's operation order (same cost matrix, same SciPy solver, same GIoU rounding)."""
        from scipy.optimize import linear_sum_assignment
        from .modules import _to_host_list
        pb = outputs["pred_boxes"].detach().cpu().numpy().astype(np.float32, copy=False)
        pc = outputs["pred_classes"].detach().cpu().numpy()
        tbl = _to_host_list([t["boxes"] for t in targets], np.float32)
        tll = _to_host_list([t["labels"] for t in targets], np.int64)
        f32 = np.float32

        def xyxy(b):
            return np.stack([b[:, 0] - f32(0.5) * b[:, 2], b[:, 1] - f32(0.5) * b[:, 3],
                             b[:, 0] + f32(0.5) * b[:, 2], b[:, 1] + f32(0.5) * b[:, 3]], -1)

        res = []
        for b, (tb, tl) in enumerate(zip(tbl, tll)):
            nb = int(n_boxes[b])
            ob, oc = pb[b, :nb], np.asarray(pc[b])
            tb, tl = np.asarray(tb, np.float32).reshape(-1, 4), np.asarray(tl).reshape(-1)
            cost = f32(self.cost_bbox) * np.abs(ob[:, None, :2] - tb[None, :, :2]).sum(-1, dtype=np.float32) \
                + f32(self.cost_class) * (oc[:nb, None].astype(np.float32) != tl[None, :].astype(np.float32)).astype(np.float32)
            rows, cols = linear_sum_assignment(cost)
            b1, b2 = xyxy(ob), xyxy(tb)
            a1, a2 = (b1[:, 2] - b1[:, 0]) * (b1[:, 3] - b1[:, 1]), (b2[:, 2] - b2[:, 0]) * (b2[:, 3] - b2[:, 1])
            wh = np.clip(np.minimum(b1[:, None, 2:], b2[None, :, 2:]) - np.maximum(b1[:, None, :2], b2[None, :, :2]), 0, None)
            inter = wh[..., 0] * wh[..., 1]
            union = a1[:, None] + a2[None, :] - inter
            wh = np.clip(np.maximum(b1[:, None, 2:], b2[None, :, 2:]) - np.minimum(b1[:, None, :2], b2[None, :, :2]), 0, None)
            area = wh[..., 0] * wh[..., 1]
            with np.errstate(divide="ignore", invalid="ignore"):
                giou = inter / union - (area - union) / area
            keep = [k for k, (i, j) in enumerate(zip(rows, cols))
                    if not (self.class_mode == "specific" and oc[i] != tl[j]) and not (giou[i, j] < giou_thresh)]
            res.append((torch.as_tensor(rows[keep], dtype=torch.int64), torch.as_tensor(cols[keep], dtype=torch.int64)))
        return res


class _PinnedRing:
    """Round-robin pinned host buffers for small per-step index uploads; a slot is rewritten only after the H2D copy that
    read it has completed (event per slot), so the host may run several steps ahead of the GPU."""

    def __init__(self, slots=8, capacity=4096):
        self.slots = [dict(buf=torch.empty(capacity, dtype=torch.int64).pin_memory(), ev=None) for _ in range(slots)]
        self.pos = 0

    def stage(self, arr: np.ndarray, device):
        slot = self.slots[self.pos]
        self.pos = (self.pos + 1) % len(self.slots)
        if slot["ev"] is not None:
            slot["ev"].synchronize()
        if slot["buf"].numel() < arr.size:
            slot["buf"] = torch.empty(2 * arr.size, dtype=torch.int64).pin_memory()
        view = slot["buf"][: arr.size].view(arr.shape)
        view.copy_(torch.from_numpy(np.ascontiguousarray(arr, dtype=np.int64)))
        out = view.to(device, non_blocking=True)
        slot["ev"] = torch.cuda.Event()
        slot["ev"].record()
        return out


def acos_linear_extrapolation(x, lo, hi):
    """util/rotation_utils.py:13-67: acos inside (lo, hi), first-order Taylor continuation outside."""
    out = torch.empty_like(x)
    up, low = x >= hi, x <= lo
    mid = ~up & ~low
    out[mid] = torch.acos(x[mid])
    for m, b in ((up, hi), (low, lo)):
        out[m] = math.acos(b) - (x[m] - b) / math.sqrt(1.0 - b * b)
    return out


def so3_log_map(R, eps=1e-4, cos_bound=1e-4):
    """util/rotation_utils.py:150-192,244-316: rotation matrices (n,3,3) -> rotation vectors (n,3).  Used by the aleatoric
    rotation loss only (a few hundred matrices; the masked assignments synchronise with the host, as the reference's do)."""
    tr = R[:, 0, 0] + R[:, 1, 1] + R[:, 2, 2]
    if bool(((tr < -1.0 - eps) | (tr > 3.0 + eps)).any()):
        raise ValueError("A matrix has trace outside valid range [-1-eps,3+eps].")
    phi = acos_linear_extrapolation((tr - 1.0) * 0.5, -(1.0 - cos_bound), 1.0 - cos_bound)
    sin = torch.sin(phi)
    fac = torch.empty_like(phi)
    ok = sin.abs() > 0.5 * eps
    fac[~ok] = 0.5 + (phi[~ok] ** 2) * (1.0 / 12)
    fac[ok] = phi[ok] / (2.0 * sin[ok])
    A = fac[:, None, None] * (R - R.permute(0, 2, 1))
    return torch.stack((A[:, 2, 1], A[:, 0, 2], A[:, 1, 0]), dim=1)


LOSS_TERMS = ("translation", "rotation", "quaternion", "silho_quaternion", "aleatoric_translation", "aleatoric_rotation")


def losses_for(rotation_mode="6d", aleatoric=False):
    """The reference's loss terms for a rotation representation / the aleatoric extension (main.py's --translation_loss /
    --rotation_loss choices)."""
    if aleatoric:
        return ("aleatoric_translation", "aleatoric_rotation")
    return ("translation", {"6d": "rotation", "quat": "quaternion", "silho_quat": "silho_quaternion"}[rotation_mode])


class SetCriterion(nn.Module):
    def __init__(self, matcher, weight_dict, losses=("translation", "rotation")):
        super().__init__()
        if any(l not in LOSS_TERMS for l in losses):
            raise NotImplementedError(f"losses {tuple(losses)}: known terms are {LOSS_TERMS}")
        self.matcher, self.weight_dict, self.losses = matcher, weight_dict, list(losses)
        self.default_terms = tuple(losses) == ("translation", "rotation")       # the pair the fused loss kernel computes

    def _gather_targets(self, targets, indices, device):
        """(batch idx, query idx, matched target translation, matched target rotation) for pose_estimation_transformer.py:
        649-668.  The matcher's indices live on the host; they travel as ONE packed int64 array through a preallocated
        pinned ring (a fresh pin_memory() per index tensor makes the host allocator register new pages every few steps,
        which stalls the GPU queue for tens of ms), and the targets are gathered with one index op per field."""
        counts = [int(t["relative_position"].shape[0]) for t in targets]
        offs = np.concatenate([[0], np.cumsum(counts)[:-1]]) if counts else np.zeros(0, np.int64)
        b = np.concatenate([np.full(len(src), i, np.int64) for i, (src, _) in enumerate(indices)])
        sq = np.concatenate([np.asarray(src, dtype=np.int64) for (src, _) in indices])
        g = np.concatenate([np.asarray(j, dtype=np.int64) + offs[i] for i, (_, j) in enumerate(indices)])
        packed = np.stack([b, sq, g])
        pos = torch.cat([t["relative_position"] for t in targets], 0)
        rot = torch.cat([t["relative_rotation"] for t in targets], 0)
        if device.type != "cuda":
            idx = torch.from_numpy(packed).to(device)
        else:
            if not hasattr(self, "_ring"):
                self._ring = _PinnedRing()
            idx = self._ring.stage(packed, device)
        gi = idx[2].to(pos.device) if pos.device != idx.device else idx[2]
        return idx[0], idx[1], pos[gi].to(device), rot[gi].to(device), idx[2], targets

    def _device_match(self, outputs, targets, n_boxes):
        """matcher.py:158-229 + the target gather of pose_estimation_transformer.py:649-668 on the device ('gt' mode): returns
        (flat query index b*Q+s, matched target translations, rotations, n_obj).  Host work: shapes (metadata) and one small
        upload of the per-image offsets; no device->host copy."""
        pb = outputs["pred_boxes"]
        dev = pb.device
        N, Q = pb.shape[:2]
        counts = [int(t["boxes"].shape[0]) for t in targets]
        n_obj = int(sum(min(int(a), c) for a, c in zip(n_boxes, counts)))
        if n_obj == 0:
            z = torch.zeros
            return z(0, dtype=torch.int64, device=dev), z((0, 3), device=dev), z((0, 3, 3), device=dev), 0
        meta = np.zeros(2 * N + 1, np.int64)
        meta[1:N + 1] = np.cumsum(counts)
        meta[N + 1:] = np.asarray(n_boxes, np.int64)
        if not hasattr(self, "_ring"):
            self._ring = _PinnedRing()
        meta_d = self._ring.stage(meta, dev).to(torch.int32)
        tb = torch.cat([t["boxes"].reshape(-1, 4) for t in targets], 0).to(dev, non_blocking=True).float().contiguous()
        tpos = torch.cat([t["relative_position"] for t in targets], 0).to(dev, non_blocking=True).float().contiguous()
        trot = torch.cat([t["relative_rotation"] for t in targets], 0).to(dev, non_blocking=True).float().contiguous()
        if not hasattr(self, "_lsa_status") or self._lsa_status.device != dev:
            self._lsa_status = torch.zeros(1, dtype=torch.int32, device=dev)
        col = torch.empty((N, Q), dtype=torch.int32, device=dev)
        ops.lsa_boxes(pb.float().contiguous(), tb, meta_d[: N + 1], meta_d[N + 1:], col, self._lsa_status, self.matcher.cost_bbox)
        # zero-filled: should the assignment kernel bail out (status != 0: non-finite costs) fewer than n_obj slots are written,
        # and the loss kernel must then still index valid rows (oversized problems never get here: see forward())
        qi = torch.zeros(n_obj, dtype=torch.int64, device=dev)
        tt = torch.zeros((n_obj, 3), dtype=torch.float32, device=dev)
        tr = torch.zeros((n_obj, 3, 3), dtype=torch.float32, device=dev)
        ops.match_gather(col, meta_d[: N + 1], tpos, trot, qi, tt, tr)
        self._last_col = col
        return qi, tt, tr, n_obj

    def device_match_status(self) -> int:
        """0 = every on-device assignment so far was solved (synchronises; call it at logging points, not per step)."""
        st = getattr(self, "_lsa_status", None)
        return 0 if st is None else int(st.item())

    def _losses(self, outputs, gathered):
        """pose_estimation_transformer.py:472-609, one entry of self.losses per term (the default pair normally takes the
        fused kernel in forward(); this is the general form)."""
        b, s, tt, tr, gi, targets = gathered
        n_obj = len(tt)
        st = outputs["pred_translation"][b, s]
        res = {}
        for name in self.losses:
            if name == "translation":
                res["loss_trans"] = torch.sqrt(((st - tt) ** 2).sum(1)).sum() / n_obj
            elif name == "aleatoric_translation":
                sa = outputs["pred_translation_aleatoric"][b, s]
                res["loss_trans"] = ((torch.exp(-sa) * torch.square(tt - st)).sum(1) + sa.sum(1)).sum() / (2 * n_obj)
            elif name in ("rotation", "aleatoric_rotation"):
                prod = torch.bmm(outputs["pred_rotation"][b, s], tr.transpose(1, 2))
                if name == "rotation":
                    trace = prod.diagonal(dim1=1, dim2=2).sum(1)
                    res["loss_rot"] = torch.acos(torch.clamp(0.5 * (trace - 1), -1 + 1e-6, 1 - 1e-6)).sum() / n_obj
                else:
                    sa = outputs["pred_rotation_aleatoric"][b, s]
                    res["loss_rot"] = ((torch.exp(-sa) * torch.square(so3_log_map(prod))).sum(1) + sa.sum(1)).sum() / (2 * n_obj)
            else:                                   # quaternion terms, [w, x, y, z], eps 1e-4
                tq = torch.cat([t["relative_quaternions"] for t in targets], 0)
                tq = tq[gi.to(tq.device)].to(st.device)
                dp = (outputs["pred_rotation"][b, s] * tq).sum(1)
                lq = -torch.log(torch.square(dp) + 1e-4) if name == "quaternion" else torch.log(1 - torch.abs(dp) + 1e-4)
                res["loss_rot"] = lq.sum() / n_obj
        return res

    def forward(self, outputs, targets, n_boxes):
        main = {k: v for k, v in outputs.items() if k not in ("aux_outputs", "enc_outputs")}
        if hasattr(self.matcher, "_cache"):
            self.matcher._cache = (None, None)      # the per-call cache must not outlive the call (static buffers are reused)
        aux_list = outputs.get("aux_outputs", [])
        for aux in aux_list:
            for k in ("_pred_boxes_host", "_tgt_boxes_host", "_pred_classes_host", "_tgt_labels_host"):
                if k in outputs:
                    aux[k] = outputs[k]
        dev = outputs["pred_translation"].device
        stacked0 = outputs.get("_stacked")
        if (self.default_terms and getattr(self.matcher, "device_assign", False) and dev.type == "cuda" and stacked0 is not None
                and stacked0[0].shape[0] == len(aux_list) + 1
                # poet_lsa_boxes solves <= 64 x 64 per image; larger problems take the host (SciPy) matcher below
                and outputs["pred_boxes"].shape[1] <= 64 and all(int(t["boxes"].shape[0]) <= 64 for t in targets)):
            # every decoder layer carries the same query boxes in 'gt' mode: ONE assignment, solved on the GPU, feeds the fused
            # loss of all layers
            from .functional import PoseLossFn
            qi, tt, tr, n_obj = self._device_match(outputs, targets, n_boxes)
            vec = PoseLossFn.apply(stacked0[0], stacked0[1], qi, tt, tr, n_obj)
            L = vec.shape[0]
            losses = LossDict({"loss_trans": vec[L - 1, 0], "loss_rot": vec[L - 1, 1]})
            for i in range(L - 1):
                losses[f"loss_trans_{i}"] = vec[i, 0]
                losses[f"loss_rot_{i}"] = vec[i, 1]
            losses.vec = vec
            return losses
        indices = self.matcher(main, targets, n_boxes)
        all_idx = [indices] + [self.matcher(aux, targets, n_boxes) for aux in aux_list]
        if self.default_terms and all(ix is indices for ix in all_idx[1:]):
            # 'gt' mode: every decoder layer gets the same assignment (same boxes), so the per-layer losses of
            # pose_estimation_transformer.py:635-674 are evaluated in ONE batched pass -- same values, ~10x fewer launches
            b, s, tt, tr = self._gather_targets(targets, indices, dev)[:4]
            n_obj = len(tt)
            stacked = outputs.get("_stacked")
            if stacked is not None and dev.type == "cuda" and stacked[0].shape[0] == len(aux_list) + 1:
                # all layers, both terms and their gradients in ONE kernel (the PyTorch form below is ~70 launches forward
                # plus as many backward, all tiny and all on the critical path between the two HIP graphs)
                from .functional import PoseLossFn
                trans_all, rot_all = stacked
                Q = trans_all.shape[2]
                vec = PoseLossFn.apply(trans_all, rot_all, b * Q + s, tt, tr, n_obj)
                L = vec.shape[0]
                losses = LossDict({"loss_trans": vec[L - 1, 0], "loss_rot": vec[L - 1, 1]})
                for i in range(L - 1):
                    losses[f"loss_trans_{i}"] = vec[i, 0]
                    losses[f"loss_rot_{i}"] = vec[i, 1]
                losses.vec = vec
                return losses
            layers = [outputs] + list(aux_list)
            st = torch.stack([o["pred_translation"] for o in layers])[:, b, s]              # (L, n_obj, 3)
            sr = torch.stack([o["pred_rotation"] for o in layers])[:, b, s]                 # (L, n_obj, 3, 3)
            lt = torch.sqrt(((st - tt) ** 2).sum(-1)).sum(-1) / n_obj
            trace = (sr * tr).sum((-1, -2))                                                 # trace(R_pred R_gt^T)
            lr = torch.acos(torch.clamp(0.5 * (trace - 1), -1 + 1e-6, 1 - 1e-6)).sum(-1) / n_obj
            losses = {"loss_trans": lt[0], "loss_rot": lr[0]}
            for i in range(len(aux_list)):
                losses[f"loss_trans_{i}"] = lt[i + 1]
                losses[f"loss_rot_{i}"] = lr[i + 1]
            return losses
        gathered, last = self._gather_targets(targets, indices, dev), indices
        losses = dict(self._losses(outputs, gathered))
        for i, (aux, ix) in enumerate(zip(aux_list, all_idx[1:])):
            if ix is not last:
                gathered, last = self._gather_targets(targets, ix, dev), ix
            losses.update({f"{k}_{i}": v for k, v in self._losses(aux, gathered).items()})
        return losses


    def total(self, loss_dict):
        """sum_k weight_dict[k] * loss_dict[k] (engine.py:62 of the reference).  With the fused loss kernel the terms are
        rows of one (L, 2) tensor and the weighted sum is two launches instead of ~20 (and as many in backward)."""
        vec = getattr(loss_dict, "vec", None)
        if vec is None:
            return sum(loss_dict[k] * self.weight_dict[k] for k in loss_dict if k in self.weight_dict)
        L = vec.shape[0]
        key = (vec.device, L)
        if getattr(self, "_wkey", None) != key:
            w = torch.zeros((L, 2), dtype=torch.float32)
            for i in range(L):
                suffix = "" if i == L - 1 else f"_{i}"
                w[i, 0] = self.weight_dict.get("loss_trans" + suffix, 0.0)
                w[i, 1] = self.weight_dict.get("loss_rot" + suffix, 0.0)
            self._w, self._wkey = w.to(vec.device), key
        return (vec * self._w).sum()


class LossDict(dict):
    """dict of differentiable scalar losses that also carries them stacked (`vec`, (L, 2)) for SetCriterion.total()."""
    vec = None


def build_weight_dict(dec_layers, t_coef=1.0, r_coef=1.0, aux=True):
    """pose_estimation_transformer.py:714,728-733 (the *_enc entries are never produced by the model)."""
    wd = {"loss_trans": t_coef, "loss_rot": r_coef}
    if aux:
        for i in range(dec_layers - 1):
            wd.update({f"loss_trans_{i}": t_coef, f"loss_rot_{i}": r_coef})
    return wd


def reduce_dict(loss_dict: Dict[str, torch.Tensor], average=True):
    """util/misc.py:168-195: all-reduce the stacked loss scalars for logging."""
    world = dist.get_world_size() if dist.is_available() and dist.is_initialized() else 1
    if world < 2:
        return loss_dict
    with torch.no_grad():
        names = sorted(loss_dict)
        vals = torch.stack([loss_dict[k].detach() for k in names])
        dist.all_reduce(vals)
        if average:
            vals = vals / world
        return dict(zip(names, vals))


def shard_indices(n_items: int, rank: int, world: int, epoch: int = 0, shuffle: bool = True):
    """Batch sharding of the reference's DistributedSampler (data_utils/samplers.py:48-66): epoch-seeded permutation,
    padded by wrap-around to a multiple of `world`, rank r takes the contiguous slice [r*n, (r+1)*n)."""
    if shuffle:
        g = torch.Generator()
        g.manual_seed(epoch)
        idx = torch.randperm(n_items, generator=g).tolist()
    else:
        idx = list(range(n_items))
    per = int(math.ceil(n_items / world))
    idx += idx[: per * world - len(idx)]
    return idx[per * rank: per * (rank + 1)]


class Trainer:
    """One training step == engine.py:55-81 (forward, loss, zero_grad, backward, clip, AdamW)."""

    def __init__(self, model: nn.Module, criterion: SetCriterion, lr=2e-4, weight_decay=1e-4, max_norm=0.1,
                 distributed: Optional[bool] = None, muon=None):
        """muon: orthogonalised updates of the weight matrices (ParamArena)."""
        self.model, self.criterion, self.max_norm = model, criterion, max_norm
        # transformer.reference_points only receives a gradient with learned reference points (else it stays outside, as
        # torch.optim.AdamW skips parameters whose .grad is None)
        exclude = () if getattr(model, "ref_points_mode", "bbox") == "learned" else ("transformer.reference_points",)
        self.arena = ParamArena(model, lr=lr, weight_decay=weight_decay, exclude=exclude, muon=muon)
        if distributed is None:
            distributed = dist.is_available() and dist.is_initialized() and (dist.get_world_size() > 1 or collectives_forced())
        self.reducer = BucketReducer(self.arena) if distributed else None
        if self.reducer is not None and self.reducer.active:
            dist.broadcast(self.arena.flat, src=0)      # DDP's initial parameter sync
            self.arena.refresh_shadow()                 # the bf16 operand copies must follow the broadcast values
            in_arena = {id(p) for _, p, _ in self.arena.entries}
            with torch.no_grad():                       # parameters outside the arena (never trained) are synced too, as DDP does
                for p in model.parameters():
                    if id(p) not in in_arena:
                        dist.broadcast(p.data, src=0)

    def step(self, samples, targets):
        with ops.pinned_stream():
            return self._step(samples, targets)

    def _step(self, samples, targets):
        set_reducer(self.reducer)
        out, n_boxes = self.model(samples, targets)
        loss_dict = self.criterion(out, targets, n_boxes)
        wd = self.criterion.weight_dict
        total = self.criterion.total(loss_dict) if hasattr(self.criterion, "total") else sum(loss_dict[k] * wd[k] for k in loss_dict if k in wd)
        self.arena.zero_grad()
        total.backward()
        if self.reducer is not None:
            self.reducer.finish()
        self.arena.step(self.max_norm)
        set_reducer(None)
        return total.detach(), loss_dict


def segment_tags(arena: ParamArena):
    """Bucket names of the arena = the points the graphed trainer cuts backward at, in backward order."""
    return [b[0] for b in arena.buckets]


def _vec_dict(vec):
    """LossDict over the rows of a stacked (L, 2) loss tensor (last row = the model output, rows 0..L-2 the auxiliary layers)."""
    L = vec.shape[0]
    d = LossDict({"loss_trans": vec[L - 1, 0], "loss_rot": vec[L - 1, 1]})
    for i in range(L - 1):
        d[f"loss_trans_{i}"] = vec[i, 0]
        d[f"loss_rot_{i}"] = vec[i, 1]
    d.vec = vec
    return d


class _Replay(torch.autograd.Function):
    """Autograd shim around the two captured graphs: forward replays the model-forward graph and hands out its static
    outputs; backward copies the loss gradients into the static grad buffers and replays backward (+ optimiser)."""

    @staticmethod
    def forward(ctx, trainer, handle):
        ctx.trainer = trainer
        trainer.g_fwd.replay()
        return (trainer.s_rot.detach(), trainer.s_trans.detach(), *[x.detach() for x in trainer.s_extra])   # (+ the aleatoric heads' outputs)

    @staticmethod
    def backward(ctx, drot, dtrans, *dextra):
        t = ctx.trainer
        t.s_drot.copy_(drot)
        t.s_dtrans.copy_(dtrans)
        for buf, g in zip(t.s_dextra, dextra):
            buf.zero_() if g is None else buf.copy_(g)
        _Replay.replay_backward(t)
        return None, None

    @staticmethod
    def replay_backward(t):
        if t.segs is None:
            t.g_bwd.replay()                 # backward + clip + AdamW in one graph (single GPU)
            return None, None
        reduce = t.reducer is not None and t.reducer.active and not getattr(t, "skip_collectives", False)   # (bench.py: exposed-collective timing)
        for g, tags in zip(t.segs, t.seg_tags):
            g.replay()
            if reduce:
                for tag in tags:
                    t.reducer.bucket_done(tag)   # event on this stream -> all-reduce of the bucket on the comm stream
        if reduce:
            t.reducer.finish()               # any range not announced yet, then this stream waits for the comm stream
        t.g_opt.replay()
        return None, None


def _stage_copy(dst: torch.Tensor, src: torch.Tensor):
    """The backbone's feature maps into the graphs' static input buffers (103 MB per step at 640x480, bs 16).  Large fp32 device tensors
    go through the library's streaming copy kernel (16-byte lanes, ~5 TB/s); torch's device-to-device copy runs at ~2.4 TB/s on this stack
    (86 us against ~40 for the largest level).  Anything else: Tensor.copy_."""
    if (src.is_cuda and src.dtype == torch.float32 and dst.dtype == torch.float32 and src.is_contiguous() and dst.is_contiguous()
            and src.numel() == dst.numel() and src.numel() >= (1 << 20) and os.environ.get("POET_STAGE_COPY", "hip") == "hip"):
        ops.cast(src, dst)
    else:
        dst.copy_(src, non_blocking=True)


class PackedBatch:
    """One batch staged ahead of its step in a GraphedTrainer's static-input layout (GraphedTrainer.pack)."""
    __slots__ = ("buf", "owner")

    def __init__(self, buf, owner):
        self.buf, self.owner = buf, owner


class GraphedTrainer(Trainer):
    """Trainer whose device work is replayed from HIP graphs (the step has ~700 kernel launches; enqueuing them from
    Python costs about as much as executing them).  Three graphs, captured after `warm` eager steps:
        g_fwd : bump the device-side dropout word; PoET.forward_core (input_proj .. heads)
        g_bwd : zero the gradient arena; the four backward programs + clip + AdamW (world == 1)
        world > 1 (default since round 4): backward is ONE graph (without the optimiser), ONE RCCL all-reduce of the flat gradient
                arena follows it, then g_opt.  POET_DP_SINGLE_COLLECTIVE=0 / segment_backward=True: one graph per gradient bucket
                (heads, decoder, every encoder layer, input_proj), each bucket's all-reduce enqueued on the comm stream right after
                its segment; bench.py times both at world > 1 and keeps the faster
        g_opt : clip + AdamW
    Host work per step: pad/pack the boxes, three small H2D copies, the matcher, the loss and its backward (eager).
    Requirements: fixed batch size / image geometry, model in train() mode for the whole run."""

    def __init__(self, model, criterion, lr=2e-4, weight_decay=1e-4, max_norm=0.1, warm=3, segment_backward=None,
                 persistent_inputs=False, muon=None):
        """persistent_inputs=True: the caller promises that the feature / mask tensors it passes are the SAME buffers on every
        step (a backbone writing into fixed outputs); they are then used as the graphs' static inputs without a copy.  The
        default keeps private static buffers and copies every step's inputs into them -- the trainer never writes into a
        tensor it does not own."""
        # the base class broadcasts the parameters and owns the bucket reducer used by the EAGER warm-up steps (without it
        # the ranks would drift apart before the graphs are captured); the captured steps all-reduce the whole arena
        # themselves (see _Replay.backward) and run with the reducer detached
        super().__init__(model, criterion, lr=lr, weight_decay=weight_decay, max_norm=max_norm, distributed=None, muon=muon)
        self.world = dist.get_world_size() if dist.is_available() and dist.is_initialized() else 1
        self.arena.world = self.world
        self.warm, self.calls, self.ready = warm, 0, False
        self.persistent_inputs = bool(persistent_inputs)
        explicit = segment_backward is not None or os.environ.get("POET_SEGMENT_BWD", "0") not in ("", "0")
        if segment_backward is None:         # backward outside the optimiser graph: needed (only) to put all-reduces between them
            segment_backward = (self.reducer is not None and self.reducer.active) or os.environ.get("POET_SEGMENT_BWD", "0") not in ("", "0")
        self.segment_backward = bool(segment_backward)
        # Default at world > 1: backward stays ONE graph (without the optimiser) and the whole gradient arena is all-reduced in ONE
        # collective behind it (BucketReducer.finish() coalesces every un-announced range).  POET_DP_SINGLE_COLLECTIVE=0 selects one
        # backward segment + one all-reduce per bucket (heads, decoder, every encoder layer, input_proj) on the comm stream instead:
        # measured on this stack (round 4, 1-rank RCCL group) the segments cost +0.19 ms per step over the single
        # collective (13.75 against 13.56 ms; 13.50 without collectives) and a kernel trace shows NO kernel of the comm queue ever
        # running concurrently with a compute-queue kernel, so the segments buy no overlap here.
        # (an explicit segment_backward=True / POET_SEGMENT_BWD=1 asks for the per-bucket segments; the environment switch wins)
        sc = os.environ.get("POET_DP_SINGLE_COLLECTIVE")
        self.single_collective = self.segment_backward and ((sc not in ("", "0")) if sc is not None else not explicit)
        if self.segment_backward and not self.single_collective and any(n.startswith("backbone.1.") for n, _, _ in self.arena.entries):
            # a learned position encoding's gradient node hangs off every encoder layer: it cannot be cut into per-bucket segments.
            # Callers that asked for them (segment_backward=True was the documented way to request the DP overlap) get the
            # single-collective mode with a warning instead of an exception
            import warnings
            warnings.warn("GraphedTrainer: learned position encoding (backbone.1.*): per-bucket backward segments are not available, "
                          "using one backward graph + one all-reduce of the gradient arena")
            self.single_collective = True
        if not self.segment_backward and self.reducer is not None and self.reducer.active:
            raise ValueError("GraphedTrainer: world > 1 needs segment_backward=True (the single backward graph contains no "
                             "all-reduce: the replicas would drift apart silently)")

    def _static_inputs(self, samples, targets):
        m = self.model
        features, _, _ = m.backbone(samples)
        boxes, classes, valid, n_boxes = m.host_queries(targets)
        return features, boxes, classes, valid, n_boxes

    def _stage_targets(self, targets, queries=False, D=None):
        """(D: destination views -- the static input buffers by default, a PackedBatch's views from pack())
        Compacted target boxes / translations / rotations and the per-image offsets + query counts into the static
        buffers the captured matcher reads (device-resident targets: device-side cat + copy; host targets: H2D).
        queries=True (targets on the device): the padded query boxes / classes / valid flags of PoET.host_queries are
        scattered into their static buffers on the device as well -- the host reads shapes only, never tensor contents, so it
        does not wait for the GPU and can run ahead of it."""
        D = self.S if D is None else D
        s_boxes, s_cls, s_valid, s_tb, s_tpos, s_trot, s_meta = (D[k] for k in ("boxes", "cls", "valid", "tb", "tpos", "trot", "meta"))
        N, Q = s_boxes.shape[:2]
        counts = [int(t["boxes"].shape[0]) for t in targets]
        n = sum(counts)
        if len(counts) != N or n > s_tb.shape[0] or max(counts, default=0) > Q:
            raise ValueError(f"GraphedTrainer: {n} targets in {len(counts)} images (max {max(counts, default=0)}) exceed the captured "
                             f"capacity ({N} images x {Q} queries; the reference assumes n <= num_queries in gt mode)")
        meta = np.zeros(2 * N + 1 + (n if queries else 0), np.int64)
        meta[1:N + 1] = np.cumsum(counts)
        meta[N + 1:2 * N + 1] = np.asarray(counts, np.int64)            # gt mode: one query per target box
        if queries and n:
            meta[2 * N + 1:] = np.concatenate([i * Q + np.arange(c, dtype=np.int64) for i, c in enumerate(counts)])
        if not hasattr(self, "_meta_ring"):
            self._meta_ring = _PinnedRing()
        meta_d = self._meta_ring.stage(meta, s_meta.device)
        s_meta.copy_(meta_d[: 2 * N + 1], non_blocking=True)
        dev = s_tb.device
        tb = None
        if n:
            def gather(key, dst, shape):                        # device-resident fp32 fields: concatenated straight into the static buffer
                parts = [t[key].reshape(shape) for t in targets]
                if all(x.is_cuda and x.dtype == dst.dtype for x in parts):
                    torch.cat(parts, 0, out=dst[:n])
                else:
                    dst[:n].copy_(torch.cat(parts, 0).to(dev, non_blocking=True), non_blocking=True)
                return dst[:n]
            tb = gather("boxes", s_tb, (-1, 4))
            gather("relative_position", s_tpos, (-1, 3))
            gather("relative_rotation", s_trot, (-1, 3, 3))
        if queries:
            s_boxes.fill_(-1.0)
            s_cls.fill_(-1)
            s_valid.zero_()
            if n:
                idx = meta_d[2 * N + 1:]
                s_boxes.view(-1, 4).index_copy_(0, idx, tb)
                s_cls.view(-1).index_copy_(0, idx, torch.cat([t["labels"].reshape(-1) for t in targets], 0).to(dev, non_blocking=True).to(s_cls.dtype))
                s_valid.view(-1).index_fill_(0, idx, 1)
        return counts

    def _capture(self, samples, targets):
        m, dev = self.model, self.arena.flat.device
        features, boxes, classes, valid, _ = self._static_inputs(samples, targets)
        # static input buffers are PRIVATE clones unless the caller registered its buffers as persistent: step() copies into
        # them, and writing into a tensor the caller owns would corrupt a batch that is stepped again later
        u8 = lambda t: t.contiguous().view(torch.uint8) if t.dtype == torch.bool else t.contiguous()
        own = (lambda t: t) if self.persistent_inputs else (lambda t: t.clone())
        self.s_feats = [own(f.tensors.contiguous()) for f in features]
        self.s_fmasks = [own(u8(f.mask)) for f in features]
        self.s_imask = own(u8(samples.mask))
        # pinned staging ring: the host may run several steps ahead of the GPU, so a slot is only rewritten after the
        # H2D copies that read it have completed (event per slot)
        self.ring = [dict(boxes=torch.from_numpy(boxes.copy()).pin_memory(), cls=torch.from_numpy(classes.copy()).pin_memory(),
                          valid=torch.from_numpy(valid.copy()).pin_memory(), ev=None) for _ in range(4)]
        self.ring_pos = 0
        self.s_boxes = self.ring[0]["boxes"].to(dev)
        self.s_cls = self.ring[0]["cls"].to(dev)
        self.s_valid = self.ring[0]["valid"].to(dev)
        self.seed_word = torch.zeros(1, dtype=torch.int32, device=dev)
        self.step_word = self.arena.step_word
        self.step_word.fill_(self.arena.step_count)
        self.handle = torch.zeros(1, device=dev, requires_grad=True)
        ops.SEED_DEV[0] = self.seed_word
        set_reducer(None)
        torch.cuda.synchronize()
        # 'gt' mode with the on-device matcher and the default loss pair: assignment + loss + their gradients are part of the
        # forward graph (no eager launches between the two replays: that stretch was 0.45 ms of the step, two thirds of it
        # idle GPU waiting for the host).  Targets travel compacted in static buffers of capacity N*Q.
        crit = self.criterion
        self.graph_loss = bool(getattr(crit, "default_terms", False) and getattr(getattr(crit, "matcher", None), "device_assign", False)
                               and getattr(m, "bbox_mode", "gt") == "gt" and hasattr(crit, "total") and getattr(m, "aux_loss", True)
                               and os.environ.get("POET_EAGER_LOSS", "0") in ("", "0")
                               # poet_lsa_boxes solves <= 64 x 64 per image (targets per image <= Q in 'gt' mode); more queries take
                               # the eager loss with the SciPy matcher instead of a captured kernel that would leave matches at -1
                               and self.s_boxes.shape[1] <= 64)
        if self.graph_loss:
            N, Q = self.s_boxes.shape[:2]
            cap = N * Q
            z = lambda *sh, dt=torch.float32: torch.zeros(sh, dtype=dt, device=dev)
            self.s_tb, self.s_tpos, self.s_trot = z(cap, 4), z(cap, 3), z(cap, 3, 3)
            self.s_meta = z(2 * N + 1, dt=torch.int32)
            self.s_col, self.s_qi = z(N, Q, dt=torch.int32), z(cap, dt=torch.int64)
            self.s_tt, self.s_tr, self.s_nobj = z(cap, 3), z(cap, 3, 3), z(1, dt=torch.int32)
            if not hasattr(crit, "_lsa_status") or crit._lsa_status.device != dev:
                crit._lsa_status = torch.zeros(1, dtype=torch.int32, device=dev)
            n_dec = len(m.transformer.decoder.layers)
            crit.total(_vec_dict(torch.zeros((n_dec, 2), device=dev)))      # builds crit._w, the (L, 2) weight table, outside the capture
        self._build_pack()
        if self.graph_loss:
            self._stage_targets(targets)
        self.g_fwd = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.g_fwd, **_CAPTURE):
            with ops.pinned_stream():
                ops.counter_add(self.seed_word, 1)
                rot, trans, hs = m.forward_core(self.s_feats, self.s_fmasks, self.s_imask, self.s_boxes, self.s_valid, self.s_cls)
                if self.graph_loss:
                    N = self.s_boxes.shape[0]
                    L = trans.shape[0]
                    ops.lsa_boxes(self.s_boxes, self.s_tb, self.s_meta[: N + 1], self.s_meta[N + 1:], self.s_col, crit._lsa_status,
                                  crit.matcher.cost_bbox)
                    ops.match_gather(self.s_col, self.s_meta[: N + 1], self.s_tpos, self.s_trot, self.s_qi, self.s_tt, self.s_tr,
                                     n_out=self.s_nobj)
                    self.s_lossvec = torch.empty((L, 2), dtype=torch.float32, device=dev)
                    gt_, gr_ = torch.empty_like(trans), torch.empty_like(rot)
                    w = crit._w
                    assert tuple(w.shape) == (L, 2), (w.shape, L)
                    # the loss weights ride in the kernel: weighted gradients and the weighted total leave it directly (no framework
                    # multiply / reduce kernels behind the loss inside the captured step)
                    self.s_total = torch.empty((), dtype=torch.float32, device=dev)
                    ops.pose_loss(trans.detach(), rot.detach(), self.s_qi, self.s_tt, self.s_tr, 0, self.s_lossvec, gt_, gr_,
                                  n_obj_dev=self.s_nobj, weights=w.contiguous().float(), total=self.s_total)
                    self.s_dtrans, self.s_drot = gt_, gr_
        self.s_rot, self.s_trans = rot, trans
        # the aleatoric heads' log-variances (pose_estimation_transformer.py:402-411) are two more static outputs of the forward graph
        al = getattr(m, "_last_aleatoric", None)
        self.s_extra = list(al) if al is not None else []
        self.s_dextra = [torch.zeros_like(x) for x in self.s_extra]
        if not self.graph_loss:
            self.s_drot, self.s_dtrans = torch.zeros_like(rot), torch.zeros_like(trans)
        self.segs = None
        if self.segment_backward:
            # Backward captured as one graph per autograd node (= one gradient bucket each: heads, decoder, every encoder layer,
            # input_proj): at replay time the bucket's RCCL all-reduce is enqueued on the comm stream right after its segment,
            # so it overlaps the remaining segments (main.py:282's DDP overlap, with graphs).  The optimiser is a last graph.
            mem, src = m.transformer._last_memory, m._last_src
            outs = m.transformer.encoder._layer_outs          # [input, out_0, ..., out_{n-1}] of the encoder layers (N*S, d)
            n_enc = len(outs) - 1
            self.segs, self.seg_tags = [], []

            def seg(fn, tags):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, pool=self.g_fwd.pool(), **_CAPTURE):
                    with ops.pinned_stream():
                        out = fn()
                self.segs.append(g)
                self.seg_tags.append(tags)
                return out

            def first():
                self.arena.zero_grad()
                return torch.autograd.grad([rot, trans, *self.s_extra], [hs], [self.s_drot, self.s_dtrans, *self.s_dextra], retain_graph=True)[0]

            from .functional import enc_bucket_tag
            if self.single_collective:
                def whole():
                    self.arena.zero_grad()
                    torch.autograd.backward([rot, trans, *self.s_extra], [self.s_drot, self.s_dtrans, *self.s_dextra])
                seg(whole, [])                    # no bucket is announced: BucketReducer.finish() reduces the whole arena at once
                n_enc = 0
            dhs = None if self.single_collective else seg(first, ["0_heads"])
            # (learned query embeddings / reference points: their nodes hang off the decoder node, not off the path to the
            # memory -- ask for those leaves too so that their backward programs run in this segment; they write into the arena
            # views themselves and hand autograd None)
            extra = [p for n, p in m.named_parameters() if n.startswith("query_embed.") or
                     (n.startswith("transformer.reference_points.") and getattr(m, "ref_points_mode", "bbox") == "learned")]
            dx = None if self.single_collective else seg(lambda: torch.autograd.grad([hs], [outs[-1]] + extra, [dhs], retain_graph=True, allow_unused=True)[0], ["1_decoder"])
            keep = [dhs, dx]
            for i in reversed(range(n_enc)):
                tags = [enc_bucket_tag(n_enc, i)] + (["2_encoder_99"] if i == 0 else [])
                if i > 0 or outs[0].requires_grad:
                    dx = seg(lambda i=i, dx=dx: torch.autograd.grad([outs[i + 1]], [outs[i]], [dx], retain_graph=True)[0], tags)
                    keep.append(dx)
                else:
                    seg(lambda dx=dx: torch.autograd.backward([outs[1]], [dx], inputs=None), tags)
            if not self.single_collective:
                seg(lambda: torch.autograd.backward([outs[0]], [dx]), ["3_input_proj"])
            self._seg_keep = keep
        else:
            self.g_bwd = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.g_bwd, pool=self.g_fwd.pool(), **_CAPTURE):
                with ops.pinned_stream():
                    self.arena.zero_grad()
                    torch.autograd.backward([rot, trans, *self.s_extra], [self.s_drot, self.s_dtrans, *self.s_dextra])
                    ops.counter_add(self.step_word, 1)
                    self.arena.step(self.max_norm, step_dev=self.step_word)
        if self.segs is not None:
            self.g_opt = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.g_opt, pool=self.g_fwd.pool(), **_CAPTURE):
                with ops.pinned_stream():
                    ops.counter_add(self.step_word, 1)
                    self.arena.step(self.max_norm, step_dev=self.step_word)
        torch.cuda.synchronize()
        self.ready = True

    def _build_pack(self):
        """Re-home every static INPUT of the graphs -- feature maps, masks, image mask, padded query boxes / classes / valid flags and
        (captured loss) the compacted targets + per-image offsets -- in ONE allocation, 256-byte aligned fields: a batch that was
        staged ahead of time in the same layout (pack()) then reaches the graphs by a single streaming copy instead of ~20 small
        launches at the head of the step.  Called once, before the capture; the attribute names keep pointing
        at the (moved) tensors.  persistent_inputs=True: the caller's feature / mask buffers stay where they are (no pack)."""
        fields = [("boxes", self.s_boxes), ("cls", self.s_cls), ("valid", self.s_valid)]
        if not self.persistent_inputs:
            fields += [(f"feat{i}", t) for i, t in enumerate(self.s_feats)] + [(f"fmask{i}", t) for i, t in enumerate(self.s_fmasks)] + [("imask", self.s_imask)]
        if self.graph_loss:
            fields += [("tb", self.s_tb), ("tpos", self.s_tpos), ("trot", self.s_trot), ("meta", self.s_meta)]
        off, self._pack_fields = 0, []
        for name, t in fields:
            nb = t.numel() * t.element_size()
            self._pack_fields.append((name, off, nb, t.dtype, tuple(t.shape)))
            off = (off + nb + 255) // 256 * 256
        self.s_pack = torch.zeros(max(off, 256), dtype=torch.uint8, device=self.s_boxes.device)
        self.S = self._pack_views(self.s_pack)
        for name, t in fields:
            self.S[name].copy_(t)
        if self.persistent_inputs:
            for i, (f, mk) in enumerate(zip(self.s_feats, self.s_fmasks)):
                self.S[f"feat{i}"], self.S[f"fmask{i}"] = f, mk
            self.S["imask"] = self.s_imask
        else:
            self.s_feats = [self.S[f"feat{i}"] for i in range(len(self.s_feats))]
            self.s_fmasks = [self.S[f"fmask{i}"] for i in range(len(self.s_fmasks))]
            self.s_imask = self.S["imask"]
        self.s_boxes, self.s_cls, self.s_valid = self.S["boxes"], self.S["cls"], self.S["valid"]
        if self.graph_loss:
            self.s_tb, self.s_tpos, self.s_trot, self.s_meta = self.S["tb"], self.S["tpos"], self.S["trot"], self.S["meta"]
        self._pack_slots, self._pack_pos = [], 0

    def _pack_views(self, buf):
        return {name: buf[off:off + nb].view(dt).view(shape) for name, off, nb, dt, shape in self._pack_fields}

    def _stage(self, D, samples, targets):
        """One batch into the destination views D (the static inputs, or a PackedBatch's): feature maps and masks as handed over by
        the backbone, the padded query boxes / classes / valid flags, and (captured loss) the compacted targets.  Returns
        (boxes, n_boxes) of PoET.host_queries on the host path, None when the targets live on the device."""
        m = self.model
        on_device = self.graph_loss and all(t["boxes"].is_cuda and t["labels"].is_cuda for t in targets)
        if on_device:
            features = m.backbone(samples)[0]
        else:
            features, boxes, classes, valid, n_boxes = self._static_inputs(samples, targets)
        for i, f in enumerate(features):
            sf, sm = D[f"feat{i}"], D[f"fmask{i}"]
            if f.tensors.data_ptr() != sf.data_ptr():
                _stage_copy(sf, f.tensors)
            if f.mask.data_ptr() != sm.data_ptr():
                sm.copy_(f.mask.view(torch.uint8) if f.mask.dtype == torch.bool else f.mask, non_blocking=True)
        im = samples.mask                                   # the extra levels' masks / valid ratios / sine encodings derive from it
        if im.data_ptr() != D["imask"].data_ptr():
            D["imask"].copy_(im.view(torch.uint8) if im.dtype == torch.bool else im, non_blocking=True)
        if on_device:
            self._stage_targets(targets, queries=True, D=D)
            return None
        slot = self.ring[self.ring_pos]
        self.ring_pos = (self.ring_pos + 1) % len(self.ring)
        if slot["ev"] is not None:
            slot["ev"].synchronize()
        slot["boxes"].copy_(torch.from_numpy(boxes)); slot["cls"].copy_(torch.from_numpy(classes)); slot["valid"].copy_(torch.from_numpy(valid))
        D["boxes"].copy_(slot["boxes"], non_blocking=True)
        D["cls"].copy_(slot["cls"], non_blocking=True)
        D["valid"].copy_(slot["valid"], non_blocking=True)
        slot["ev"] = torch.cuda.Event()
        slot["ev"].record()
        if self.graph_loss:
            self._stage_targets(targets, D=D)
        return boxes, n_boxes

    def pack(self, samples, targets):
        """Stage one batch AHEAD of its step: into a device buffer laid out like the graphs' static input area (a ring of two, so
        batch i + 1 can be packed -- by a prefetcher, on its own stream, under the step of batch i -- while batch i is consumed).
        `step(packed)` then costs one streaming copy.  The captured-loss mode only ('gt' queries, device matcher): the eager
        loss needs the host-side query assembly of its own batch.  Returns a PackedBatch; valid until two more pack() calls."""
        if not self.ready:
            raise RuntimeError("GraphedTrainer.pack: call step(samples, targets) until the graphs are captured (warm + 1 steps) first")
        if not self.graph_loss or self.persistent_inputs:
            raise NotImplementedError("GraphedTrainer.pack: needs the captured loss ('gt' queries, device matcher) and private static inputs")
        if len(self._pack_slots) < 2:
            self._pack_slots.append(torch.empty_like(self.s_pack))
        buf = self._pack_slots[self._pack_pos]
        self._pack_pos = (self._pack_pos + 1) % 2
        self._stage(self._pack_views(buf), samples, targets)
        return PackedBatch(buf, self)

    def step(self, samples, targets=None):
        self.calls += 1
        if isinstance(samples, PackedBatch):
            if samples.owner is not self or not self.ready:
                raise ValueError("GraphedTrainer.step: a PackedBatch belongs to the trainer that packed it")
            n4 = self.s_pack.numel() // 4
            ops.cast(samples.buf[: n4 * 4].view(torch.float32), self.s_pack[: n4 * 4].view(torch.float32))      # ONE streaming copy (fields are 256-B aligned)
            self.g_fwd.replay()
            _Replay.replay_backward(self)
            return self.s_total.clone(), _vec_dict(self.s_lossvec.clone())
        if not self.ready:
            if self.calls <= self.warm:
                return super().step(samples, targets)        # eager warm-up (also fills every lazy cache)
            self._capture(samples, targets)
        m = self.model
        staged = self._stage(self.S, samples, targets)
        if staged is None:                                   # targets on the device (captured loss)
            self.g_fwd.replay()
            _Replay.replay_backward(self)
            return self.s_total.clone(), _vec_dict(self.s_lossvec.clone())      # (the static buffers are overwritten by the next replay)
        boxes, n_boxes = staged
        if self.graph_loss:
            self.g_fwd.replay()
            _Replay.replay_backward(self)
            vec = self.s_lossvec.clone()                         # the static buffers are overwritten by the next replay
            return self.s_total.clone(), _vec_dict(vec)
        rot, trans, *extra = _Replay.apply(self, self.handle)
        m._last_aleatoric = tuple(extra) if extra else None
        out = m.make_outputs(rot, trans, self.s_boxes, self.s_cls, boxes)
        loss_dict = self.criterion(out, targets, n_boxes)
        wd = self.criterion.weight_dict
        total = self.criterion.total(loss_dict) if hasattr(self.criterion, "total") else sum(loss_dict[k] * wd[k] for k in loss_dict if k in wd)
        total.backward()
        return total.detach(), loss_dict


class GraphedInference:
    """Inference (engine.py:96-184's forward; bbox_mode 'backbone' or 'gt'): the device part of `PoET.forward` is captured
    once as a HIP graph and replayed per call -- at batch 1 the eager launch sequence (~250 launches) costs more host time
    than the kernels take.  Per call on the host: the query assembly (detector rows -> padded boxes / classes), three small
    H2D copies, one graph launch.  Fixed batch size / image geometry; the feature maps are read in place when the backbone
    hands over the same buffers every call, copied into the captured ones otherwise."""

    def __init__(self, model: nn.Module, warm: int = 1):
        self.model, self.warm, self.calls, self.ready = model.eval(), warm, 0, False
        self._pack_heads()

    def _pack_heads(self):
        """Re-home the pose-head parameters of every decoder layer in one buffer per head family, equally spaced: the heads
        then run as batched launches (functional.HeadsFn) exactly as they do on the trainer's flat arena.  Values, names and
        state_dict are untouched; only `.data` moves."""
        for fam in ("translation_head", "rotation_head"):
            heads = getattr(self.model, fam, None)
            if heads is None or len(heads) < 2:
                continue
            per = [[p for _, p in h.named_parameters()] for h in heads]
            if any(p.dtype != torch.float32 or not p.is_cuda for ps in per for p in ps):
                continue
            sizes = [(p.numel() + 63) // 64 * 64 for p in per[0]]           # 256-byte aligned slots
            T = sum(sizes)
            buf = torch.empty(len(per) * T, dtype=torch.float32, device=per[0][0].device)
            with torch.no_grad():
                for i, ps in enumerate(per):
                    off = i * T
                    for p, sz in zip(ps, sizes):
                        view = buf[off: off + p.numel()].view(p.shape)
                        view.copy_(p.data)
                        p.data = view
                        off += sz

    def _inputs(self, samples, targets):
        m = self.model
        features, _, pred_objects = m.backbone(samples)
        if m.bbox_mode == "backbone":
            hw = samples.tensors.shape[-2:] if getattr(samples, "tensors", None) is not None else samples.mask.shape[-2:]
            q = m.host_queries_backbone(pred_objects, hw)
        else:
            q = m.host_queries(targets)
        return (features,) + tuple(q)

    @torch.no_grad()
    def __call__(self, samples, targets=None):
        m = self.model
        self.calls += 1
        if not self.ready and self.calls <= self.warm:
            return m(samples, targets)                        # eager warm-up (fills the lazy caches)
        features, boxes, classes, valid, n_boxes = self._inputs(samples, targets)
        u8 = lambda t: t.contiguous().view(torch.uint8) if t.dtype == torch.bool else t.contiguous()
        if not self.ready:
            dev = features[0].tensors.device
            self.s_feats = [f.tensors.contiguous().clone() for f in features]
            self.s_fmasks = [u8(f.mask).clone() for f in features]
            self.s_imask = u8(samples.mask).clone()
            self.pin = [torch.from_numpy(a.copy()).pin_memory() for a in (boxes, classes, valid)]
            self.s_boxes, self.s_cls, self.s_valid = (p.to(dev) for p in self.pin)
            self.ev = None
            torch.cuda.synchronize()
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph, **_CAPTURE):
                with ops.pinned_stream():
                    self.s_rot, self.s_trans, _ = m.forward_core(self.s_feats, self.s_fmasks, self.s_imask, self.s_boxes,
                                                                 self.s_valid, self.s_cls)
            self.ready = True
        for f, sf, sm in zip(features, self.s_feats, self.s_fmasks):
            if f.tensors.data_ptr() != sf.data_ptr():
                _stage_copy(sf, f.tensors)
            sm.copy_(u8(f.mask), non_blocking=True)
        self.s_imask.copy_(u8(samples.mask), non_blocking=True)
        if self.ev is not None:
            self.ev.synchronize()                             # the previous call's uploads have left the pinned buffers
        for p, a in zip(self.pin, (boxes, classes, valid)):
            p.copy_(torch.from_numpy(a))
        self.s_boxes.copy_(self.pin[0], non_blocking=True)
        self.s_cls.copy_(self.pin[1], non_blocking=True)
        self.s_valid.copy_(self.pin[2], non_blocking=True)
        self.ev = torch.cuda.Event()
        self.ev.record()
        self.graph.replay()
        return m.make_outputs(self.s_rot, self.s_trans, self.s_boxes, self.s_cls, boxes), n_boxes
