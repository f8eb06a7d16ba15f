"""Training the classifier end of a loaded model on labelled clips, everything before it frozen: the head Linear and, for the
two-stream transformer, the encoder's last LayerNorm -- what adapting the recogniser to another vocabulary or signer needs.

    model = AslClipModel("resnet18_mean"); model.load_state_dict(sd)
    tuner = HeadTuner(model, lambda ps: torch.optim.AdamW(ps, lr=1e-3), max_norm=1.0)
    for clips, target in batches:
        loss = tuner.step(clips, target)          # 0-d tensor on the GPU; nothing is waited for
    sd.update(tuner.state_dict())                 # and model(clips) already computes with the tuned weights

A step runs the frozen forward, then the operators of ``training``: LayerNorm forward and backward (transformer), the Linear
and its softmax cross entropy with all gradients in one call, and clipping by the global norm; the update itself is the
optimizer's, on fp32 weights in place.
"""
from __future__ import annotations

import ctypes as C
from typing import Callable, Dict, List, Optional

import torch

from . import _lib as L
from . import training
from .model import AslClipModel


class HeadTuner:
    def __init__(self, model: AslClipModel, optimizer: Callable[[List[torch.Tensor]], torch.optim.Optimizer],
                 max_norm: Optional[float] = 1.0, label_smoothing: float = 0.0, ignore_index: int = -100):
        self.model, self.max_norm = model, max_norm
        self.params: Dict[str, torch.Tensor] = model.head_parameters()
        self.optimizer = optimizer(list(self.params.values()))
        self._how = dict(ignore_index=ignore_index, label_smoothing=label_smoothing)
        names = list(self.params)
        self._fc_w, self._fc_b = self.params[names[0]], self.params[names[1]]
        self._norm = [self.params[n] for n in names[2:]]           # the last LayerNorm's weight and bias, if it is trained
        self.grad_norm: Optional[torch.Tensor] = None              # of the last step, before clipping

    def _here(self):
        """the forward launches on the current device's stream, the training operators on their tensors': one and the same here"""
        return torch.cuda.device(self._fc_w.device)

    def _features(self, clips, keypoints):
        """(features of the Linear [B, F], and for the transformer what the norm's backward needs)"""
        if any(p is not self.params.get(n) for n, p in self.model.head_parameters().items()):
            raise RuntimeError("the model's weights were loaded anew: build another HeadTuner for them")
        x = self.model.head_input(clips, keypoints)
        if not self._norm:
            return x, None
        B, T = clips.shape[:2]
        y, mean, rstd = training.layer_norm_fwd(x, *self._norm)
        pooled = torch.empty(B, x.shape[1], dtype=torch.float32, device=x.device)
        stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
        L.check(L.lib.asl_mean_t_f32(C.c_void_p(y.data_ptr()), B, T, x.shape[1], C.c_void_p(pooled.data_ptr()), stream), "mean_t")
        return pooled, (x, mean, rstd, T)

    @torch.no_grad()
    def gradients(self, clips: torch.Tensor, target: torch.Tensor, keypoints: Optional[torch.Tensor] = None):
        """(loss, {name: gradient}) of the mean cross entropy of clips [B,T,3,S,S] against target int64 [B]"""
        with self._here():
            feats, saved = self._features(clips, keypoints)
            loss, dfeats, dw, db = training.linear_cross_entropy_grad(feats, self._fc_w, target.to(feats.device), self._fc_b, **self._how)
            grads = [dw, db]
            if saved is not None:
                x, mean, rstd, T = saved
                dy = (dfeats / T)[:, None].expand(-1, T, -1).reshape(x.shape)      # the mean over T hands every frame its share
                grads += training.layer_norm_bwd(dy, x, self._norm[0], mean, rstd)[1:]
            return loss, dict(zip(self.params, grads))

    @torch.no_grad()
    def loss(self, clips: torch.Tensor, target: torch.Tensor, keypoints: Optional[torch.Tensor] = None) -> torch.Tensor:
        """the mean loss alone (validation)"""
        with self._here():
            feats, _ = self._features(clips, keypoints)
            return training.linear_cross_entropy_fwd(feats, self._fc_w, target.to(feats.device), self._fc_b, **self._how)[0]

    @torch.no_grad()
    def step(self, clips: torch.Tensor, target: torch.Tensor, keypoints: Optional[torch.Tensor] = None) -> torch.Tensor:
        """one update; returns the loss before it"""
        loss, grads = self.gradients(clips, target, keypoints)
        if self.max_norm is not None:
            with self._here():
                self.grad_norm = training.clip_grads(list(grads.values()), self.max_norm)
        for name, p in self.params.items():
            p.grad = grads[name]
        self.optimizer.step()
        for p in self.params.values():
            p.grad = None
        return loss

    def state_dict(self) -> Dict[str, torch.Tensor]:
        """the tuned weights under the names and shapes that load_state_dict takes, copied to the CPU"""
        from .spec import param_shapes
        shapes = param_shapes(self.model.spec)
        return {n: p.detach().cpu().clone().reshape(shapes[n]) for n, p in self.params.items()}
