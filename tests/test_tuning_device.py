"""CPU: a tuner's calls run with its model's device as the current one, whichever the caller's is: the frozen forward launches on
the current device's stream, the training operators on that of their tensors, and both have to be the same."""
import pytest
import torch


class _Device:
    """stands for torch.cuda.device and records what is entered"""
    current = []

    def __init__(self, device):
        self.device = device

    def __enter__(self):
        _Device.current.append(self.device)

    def __exit__(self, *exc):
        _Device.current.pop()


class _Model:
    def __init__(self):
        self.ps = {"fc.weight": torch.zeros(5, 4), "fc.bias": torch.zeros(5)}
        self.seen = []

    def head_parameters(self):
        return dict(self.ps)

    def head_input(self, clips, keypoints=None):
        self.seen.append(list(_Device.current))
        return torch.zeros(clips.shape[0], 4)


@pytest.mark.parametrize("call", ["gradients", "loss", "step"])
def test_calls_run_on_the_models_device(monkeypatch, call):
    from video_asl_recognition_amd import training, tuning
    model, clips, target = _Model(), torch.zeros(2, 3, 3, 8, 8), torch.zeros(2, dtype=torch.int64)
    where = []

    def grad(x, w, t, b, **how):
        where.append(list(_Device.current))
        return torch.zeros(()), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    monkeypatch.setattr(training, "linear_cross_entropy_grad", grad)
    monkeypatch.setattr(training, "linear_cross_entropy_fwd", lambda *a, **k: grad(*a, **k)[:2])
    monkeypatch.setattr(training, "clip_grads", lambda grads, m: where.append(list(_Device.current)) or torch.zeros(()))
    monkeypatch.setattr(torch.cuda, "device", _Device)
    tuner = tuning.HeadTuner(model, lambda ps: torch.optim.SGD(ps, lr=0.1))
    getattr(tuner, call)(clips, target)
    device = model.ps["fc.weight"].device
    assert model.seen and all(s and s[-1] == device for s in model.seen)
    assert where and all(s and s[-1] == device for s in where) and not _Device.current
