"""Answers with a trained Mamba-2 language model (mamba_lm.py) over the C ABI: greedy and beam search over packed prompts,
every computation a ``launch_*`` call on one stream.

Per layer and sequence three states are kept: the last d_conv - 1 inputs of the convolution's x columns, those of its B and C
columns (r16), and the scan's [heads, headdim, d_state] (r32).  A batch of prompts of any lengths goes through the layers once,
packed row behind row; after it every new token costs one pass over the weights and the states:

    prompt   embedding, then per layer: rmsnorm, projection, convolution and scan that begin each sequence, gate and norm,
             projection with the residual; logits of each prompt's last row
    token    the same for one row per beam, going on from the states
    search   launch_beam_select over the logits, launch_reorder_states where there are several beams

Scores are sums of log-probabilities.  From the third token on a step is one graph launch.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np

from .mamba_lm import ALIGN, LMConfig
from .runtime import Stream, launch, lib


def load_weights(cfg: LMConfig, prefix: str):
    """The weights of a checkpoint written by ``MambaLM.save`` (name -> float32 array)."""
    out = {}
    for idx, (name, shape) in enumerate(cfg.param_shapes()):
        a = np.fromfile(f"{prefix}_{idx}", dtype=np.float32)
        if a.size != math.prod(shape):
            raise ValueError(f"{prefix}_{idx}: expected {math.prod(shape)} values for {name}, found {a.size}")
        out[name] = a.reshape(shape)
    return out


class Generator:
    """Keeps the weights, the states of `sequences` sequences (prompts times beams) and buffers for prompts of `max_rows` tokens in all.

    weights: name -> array (`mamba_lm.init_weights`, `load_weights`), or a `MambaLM`, whose buffers are used as they are at each call.

    Everything runs on `stream` (a model's own, or one that the generator opens).  `prompt` and `token` take their turn behind what torch's current
    stream holds when they are called, and that stream waits for them: tokens and logits need no synchronising there.  Work on other streams is the
    caller's to order.  `search` waits for its results.  Call `release()` before the object goes."""

    def __init__(self, cfg: LMConfig, weights, sequences: int, max_rows: int, stream: Stream | None = None):
        if sequences < 1 or max_rows < 1:
            raise ValueError("at least one sequence and one row")
        if cfg.d_state > 256 or not 2 <= cfg.d_conv <= 4:
            raise ValueError("d_state is 256 at most, d_conv 2 to 4")
        import torch
        self.cfg, self.sequences, self.max_rows = cfg, sequences, max_rows
        model = weights if hasattr(weights, "w16") else None
        if model is not None and model.cfg.param_shapes() != cfg.param_shapes():
            raise ValueError("the model has another configuration")
        if model is not None and stream is not None and stream is not model.stream:
            raise ValueError("a model's buffers are used on the model's stream")
        self._own_stream = stream is None and model is None
        self.stream = stream if stream is not None else model.stream if model is not None else Stream()
        self._lib = lib()
        if model is not None:
            self.offsets, self.w16, self.w32 = model.offsets, model.w16, model.w32
        else:
            self.offsets, off = {}, 0
            for name, shape in cfg.param_shapes():
                self.offsets[name] = (off, shape)
                off += (math.prod(shape) + ALIGN - 1) // ALIGN * ALIGN
            host = torch.zeros(off, dtype=torch.float32)
            for name, (o, shape) in self.offsets.items():
                if tuple(np.shape(weights[name])) != tuple(shape):
                    raise ValueError(f"{name}: shape {np.shape(weights[name])} instead of {shape}")
                host[o:o + math.prod(shape)] = torch.from_numpy(np.ascontiguousarray(weights[name], dtype=np.float32)).reshape(-1)
            self.w32 = host.cuda()
            self.w16 = torch.empty(off, dtype=torch.float16, device="cuda")
        rows, c, gn = max(max_rows, sequences), cfg, cfg.ngroups * cfg.d_state
        f16 = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
        self.conv_x, self.conv_bc = f16(c.n_layer, sequences, c.d_conv - 1, c.d_inner), f16(c.n_layer, sequences, c.d_conv - 1, 2 * gn)
        self.ssm = torch.zeros(c.n_layer, sequences, c.heads, c.headdim, c.d_state, dtype=torch.float32, device="cuda")
        self.h = (f16(rows, c.d_model), f16(rows, c.d_model))
        self.xn, self.zx, self.xs, self.bc, self.y, self.un = (f16(rows, n) for n in (c.d_model, c.d_in_proj, c.d_inner, 2 * gn, c.d_inner, c.d_inner))
        self.last, self.hn, self.logits = f16(sequences, c.d_model), f16(sequences, c.d_model), f16(sequences, c.vocab)
        self.ids, self.starts, self.slots, self.last_rows = i32(rows), i32(sequences + 1), i32(sequences), i32(sequences)
        self.scores = torch.zeros(sequences, dtype=torch.float32, device="cuda")
        self.finished, self.parents, self.tokens = i32(sequences), i32(sequences), i32(sequences)
        self.scratch = None
        self._graph, self._graph_of = None, None
        torch.cuda.synchronize()      # torch made these on its own stream
        if model is None:
            self._lib.launch_convert_r32_r16(C.c_void_p(self.w32.data_ptr()), C.c_void_p(self.w16.data_ptr()), self.w16.numel(), self.stream.ctx)

    # ------------------------------------------------------------------ the layers
    def _p(self, buf, name):
        return buf.data_ptr() + self.offsets[name][0] * buf.element_size()

    def _L(self, name, *args):
        import torch
        launch(name, torch.float16, *args, self.stream)

    def _room(self, nbytes):
        """Scratch of the scan and the selection, which run one after the other."""
        import torch
        if self.scratch is None or self.scratch.numel() < nbytes:
            self._drop_graph()      # it holds the old address
            self.stream.sync()
            self.scratch = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
            torch.cuda.current_stream().synchronize()      # torch hands out memory that its own stream may still be at work on

    def _behind_torch(self):
        import torch
        self.stream.torch_stream().wait_stream(torch.cuda.current_stream())

    def _before_torch(self):
        import torch
        torch.cuda.current_stream().wait_stream(self.stream.torch_stream())

    def _upload(self, dst, values):
        a = np.ascontiguousarray(values, dtype=np.int32)
        self._lib.mpMemcpyHtoD(C.c_void_p(dst.data_ptr()), C.c_void_p(a.ctypes.data), a.nbytes, self.stream.ctx)
        return a

    def _layers(self, ids, rows, prompts):
        """The residual stream behind the last layer for `rows` rows: `prompts` packed sequences, or one new token of each sequence (0)."""
        c, W, W32 = self.cfg, self.w16, self.w32
        di, gn2, H, P = c.d_inner, 2 * c.ngroups * c.d_state, c.heads, c.headdim
        shape = (H, P, c.d_state, c.ngroups)
        h, other = self.h
        self._L("embedding", self._p(W, "embedding"), ids, h, rows, c.d_model, c.vocab)
        zx = self.zx.data_ptr()
        bc, cc = self.bc.data_ptr(), self.bc.data_ptr() + gn2       # (gn2 / 2 columns of two bytes)
        for i in range(c.n_layer):
            p = f"layers.{i}."
            self._L("rmsnorm_ij_j", h, self._p(W, p + "norm_w"), c.eps, self.xn, None, rows, c.d_model)
            self._L("inner_product_ij_jk_ik", self.xn, self._p(W, p + "in_proj"), 1.0, self.zx, 0.0, rows, c.d_model, c.d_in_proj)
            conv_w, conv_b = self._p(W, p + "conv_w"), self._p(W, p + "conv_b")
            # x into a tensor of its own (the gate reads it whole), B and C side by side
            for first, n, states, out in ((0, di, self.conv_x[i], self.xs), (di, gn2, self.conv_bc[i], self.bc)):
                ins = (zx + 2 * (di + first), c.d_in_proj, conv_w + 2 * first * c.d_conv, conv_b + 2 * first, states)
                if prompts:
                    self._L("causal_conv1d_silu_prompt", *ins, self.slots, None, self.starts, out, n, prompts, rows, self.sequences, n, c.d_conv)
                else:
                    self._L("causal_conv1d_silu_token", *ins, None, out, n, rows, self.sequences, n, c.d_conv)
            ins = (self.xs, di, zx + 2 * (di + c.conv_dim), c.d_in_proj, self._p(W32, p + "dt_bias"), self._p(W32, p + "A_log"), bc, cc, gn2, self.ssm[i])
            if prompts:
                self._L("ssd_scan_prompt", *ins, self.slots, None, self.starts, self.y, di, self.scratch, prompts, rows, self.sequences, *shape)
            else:
                self._L("ssd_scan_token", *ins, None, self.y, di, rows, self.sequences, *shape)
            self._L("ssd_gate_rmsnorm", self.y, self.xs, self._p(W32, p + "D"), zx, c.d_in_proj, self._p(W, p + "gnorm_w"), c.eps, self.un, None, rows, H, P)
            self._L("linear_ij_jk_ik_ik", self.un, self._p(W, p + "out_proj"), h, 1.0, other, 0.0, rows, di, c.d_model)
            h, other = other, h
        return h

    def _head(self, h, n):
        c, W = self.cfg, self.w16
        self._L("rmsnorm_ij_j", h, self._p(W, "normf_w"), c.eps, self.hn, None, n, c.d_model)
        self._L("inner_product_ij_kj_ik", self.hn, self._p(W, "embedding"), 1.0, self.logits, 0.0, n, c.d_model, c.vocab)

    # ------------------------------------------------------------------ prompts and tokens
    def _check(self, prompts, beams):
        n = len(prompts) * beams
        if not 1 <= beams <= 32:
            raise ValueError("1 to 32 beams")
        if beams > self.cfg.vocab:
            raise ValueError("more beams than tokens")
        if not prompts or n > self.sequences:
            raise ValueError(f"{len(prompts)} prompts of {beams} beams: this generator keeps {self.sequences} sequences")
        lens = [len(p) for p in prompts]
        if min(lens) < 1:
            raise ValueError("a prompt has at least one token")
        if sum(lens) > self.max_rows:
            raise ValueError(f"{sum(lens)} tokens of prompts: this generator has buffers for {self.max_rows}")
        ids = np.concatenate([np.asarray(p) for p in prompts])
        if ids.dtype.kind not in "iu" or ids.min() < 0 or ids.max() >= self.cfg.vocab:
            raise ValueError("tokens are whole numbers in [0, vocab)")
        return lens, ids

    def prompt(self, prompts, beams: int = 1):
        """Takes the prompts in; returns the r16 logits [len(prompts) * beams, vocab] behind their last tokens (a device buffer that the next
        call overwrites; torch's current stream waits for them).  The state of prompt i lies in sequence i * beams."""
        lens, ids = self._check(prompts, beams)
        self._behind_torch()      # it may be reading the last logits
        n = len(prompts) * beams
        starts = np.concatenate([[0], np.cumsum(lens)])
        keep = [self._upload(self.ids, ids), self._upload(self.starts, starts), self._upload(self.slots, np.arange(len(prompts)) * beams),
                self._upload(self.last_rows, np.repeat(starts[1:] - 1, beams))]
        rows = int(starts[-1])
        self._room(self._lib.mpSsdScanPromptScratchBytes(0, len(prompts), rows, self.cfg.heads, self.cfg.headdim, self.cfg.d_state, self.cfg.ngroups))
        h = self._layers(self.ids, rows, len(prompts))
        self._L("embedding", h, self.last_rows, self.last, n, self.cfg.d_model, rows)      # rows gathered by their numbers
        self._head(self.last, n)
        del keep
        self._before_torch()
        return self.logits[:n]

    def token(self, tokens):
        """One new token (int32, device) of each of the first len(tokens) sequences; returns their logits (see `prompt`).  The tokens are read
        behind what torch's current stream holds now."""
        import torch
        n = tokens.numel()
        if not 1 <= n <= self.sequences or tokens.dtype != torch.int32 or not tokens.is_cuda or not tokens.is_contiguous():
            raise ValueError("tokens: up to `sequences` contiguous int32 values on the device")
        self._behind_torch()
        self._head(self._layers(tokens, n, 0), n)
        self._before_torch()      # (so the caller may let go of the tokens too: torch reuses their memory behind this)
        return self.logits[:n]

    # ------------------------------------------------------------------ search
    def _select(self, batch, beams, eos):
        self._L("beam_select", self.logits, self.cfg.vocab, self.scores, self.finished, eos, self.scores, self.parents, self.tokens, self.finished,
                self.scratch, batch, beams, self.cfg.vocab, beams)

    def _go_on(self, batch, beams, eos):
        """The states follow the beams, their tokens go through the layers, the next ones are chosen."""
        import torch
        c = self.cfg
        if beams > 1:
            for states, dtype in ((self.conv_x, torch.float16), (self.conv_bc, torch.float16), (self.ssm, torch.float32)):
                launch("reorder_states", dtype, states, None, self.parents, c.n_layer, batch, beams, self.sequences, states[0, 0].numel(), self.stream)
        n = batch * beams
        self._head(self._layers(self.tokens, n, 0), n)
        self._select(batch, beams, eos)

    def search(self, prompts, new_tokens: int, beams: int = 1, eos: int | None = None):
        """The `beams` best continuations of every prompt that a beam search finds (beams = 1: greedy), best first:
        [[(tokens, score), ...], ...].  A continuation ends with `eos`, which it includes, or after `new_tokens` tokens."""
        import torch
        if new_tokens < 1:
            raise ValueError("at least one new token")
        if eos is not None and not 0 <= eos < self.cfg.vocab:
            raise ValueError("eos is a token")
        self._check(prompts, beams)
        batch, n, end = len(prompts), len(prompts) * beams, self.cfg.vocab if eos is None else eos
        self._room(self._lib.mpBeamSelectScratchBytes(0, batch, beams, self.cfg.vocab, beams))
        history = torch.empty(2, new_tokens, n, dtype=torch.int32, device="cuda")
        torch.cuda.current_stream().synchronize()
        self.prompt(prompts, beams)
        first = np.where(np.arange(n) % beams == 0, 0.0, -np.inf).astype(np.float32)      # one beam to begin with
        self._upload(self.scores, first.view(np.int32))
        self._upload(self.finished, np.zeros(n))
        self._select(batch, beams, end)
        for t in range(new_tokens):
            for k, buf in enumerate((self.tokens, self.parents)):      # whole numbers of four bytes: the copy is bit-exact
                self._lib.launch_copy_r32(C.c_void_p(buf.data_ptr()), C.c_void_p(history[k, t].data_ptr()), n, self.stream.ctx)
            if t + 1 == new_tokens:
                break
            what = (batch, beams, end)
            if t == 0:
                self._go_on(*what)      # also whatever its kernels set up on their first launch
                continue
            if self._graph_of != what:
                self._drop_graph()
                self._lib.mpGraphBeginCapture(self.stream.ctx)
                self._go_on(*what)
                self._graph, self._graph_of = self._lib.mpGraphEndCapture(self.stream.ctx), what
            self._lib.mpGraphLaunch(self._graph, self.stream.ctx)
        self.stream.sync()
        tokens, parents = history.cpu().numpy().reshape(2, new_tokens, batch, beams)
        scores = self.scores[:n].cpu().numpy().reshape(batch, beams)
        out = []
        for b in range(batch):
            found = []
            for j in range(beams):
                if scores[b, j] == -np.inf:      # fewer continuations than beams
                    continue
                line, at = [], j
                for t in reversed(range(new_tokens)):
                    line.append(int(tokens[t, b, at]))
                    at = parents[t, b, at]
                line.reverse()
                if eos is not None and eos in line:
                    line = line[:line.index(eos) + 1]
                found.append((line, float(scores[b, j])))
            out.append(found)
        return out

    def _drop_graph(self):
        if self._graph is not None:
            self.stream.sync()
            self._lib.mpGraphDestroy(self._graph)
        self._graph, self._graph_of = None, None

    def release(self):
        """Destroy the captured graph and the generator's own stream; the device buffers go with the object."""
        self.stream.sync()
        self._drop_graph()
        if self._own_stream:
            self.stream.close()
