"""The training step with a teacher, on the CPU reference path and through both entry points."""
import pytest
import torch

from test_cli_cpu import _run, ROOT


def _step(distill, steps=3):
    from pytorch_cifar_amd import models
    from pytorch_cifar_amd.data.loader import DeviceLoader
    from pytorch_cifar_amd.data.synthetic import synthetic_cifar10
    from pytorch_cifar_amd.engine.optim import SGD
    from pytorch_cifar_amd.engine.trainer import TrainStep

    torch.manual_seed(0)
    net = models.LeNet()
    opt = SGD(net.parameters(), lr=0.05, momentum=0.9)
    imgs, labs = synthetic_cifar10(64, seed=1)
    loader = DeviceLoader(imgs, labs, 16, "cpu", crop_pad=0, flip=False, drop_last=True, seed=0)
    step = TrainStep(net, opt, loader, 16, distill=distill)
    loader.set_epoch(0)
    losses, batches = [], []
    before = [p.detach().clone() for p in net.parameters()]
    for i, idx in enumerate(loader.batch_indices()):
        if i == steps:
            break
        batches.append(idx)
        losses.append(float(step(idx).detach()))
    return net, before, losses, step, batches, loader


def test_step_is_the_loss_and_its_gradient():
    """One step against the loss written out by autograd on the same weights and batch."""
    from pytorch_cifar_amd import models
    from pytorch_cifar_amd.engine.distillation import Distillation
    from pytorch_cifar_amd.nn import functional as PF

    torch.manual_seed(7)
    teacher = models.LeNet()
    d = Distillation(teacher, k=4, temperature=3.0, alpha=0.7, tail=True)
    assert not teacher.training and not any(p.requires_grad for p in teacher.parameters())
    net, before, losses, step, batches, loader = _step(d, steps=1)
    x, y = loader.make_batch(batches[0])
    fresh = models.LeNet()
    with torch.no_grad():
        for p, v in zip(fresh.parameters(), before):
            p.copy_(v)
    top = PF.top_logits(teacher(x), 4, 3.0)
    loss = PF.distill_loss(fresh(x), top, y, temperature=3.0, alpha=0.7, tail=True)
    assert losses[0] == loss.item()
    loss.backward()
    for p, q, v in zip(net.parameters(), fresh.parameters(), before):
        # (the update rounds the product and the sum, or the sum alone)
        want = v.double() - 0.05 * q.grad.double()
        assert ((p.double() - want).abs() <= 2.0 ** -23 * (want.abs() + 0.05 * q.grad.abs())).all()
    # the metrics are the labels' alone
    ce = torch.nn.functional.cross_entropy(fresh(x), y)
    assert abs(step.metrics[0].item() - ce.item()) <= 1e-6 * abs(ce.item()) and step.metrics[2].item() == 16


def test_the_teacher_stands_still():
    from pytorch_cifar_amd import models
    from pytorch_cifar_amd.engine.distillation import Distillation

    torch.manual_seed(7)
    teacher = models.ResNet18()
    state = {k: v.clone() for k, v in teacher.state_dict().items()}
    _step(Distillation(teacher))
    assert all(torch.equal(v, state[k]) for k, v in teacher.state_dict().items())


def test_without_a_teacher_nothing_changes():
    assert _step(None)[2] == _step(None)[2]


def _teacher_ckpt(path, name="LeNet"):
    from pytorch_cifar_amd import models
    from pytorch_cifar_amd.engine.checkpoint import save_checkpoint

    torch.manual_seed(3)
    return save_checkpoint(str(path / "teacher.pth"), models.build_model(name), 50.0, 1)


def test_main_py_with_a_teacher(tmp_path):
    base = [f"{ROOT}/main.py", "--cpu", "--synthetic", "--synthetic_size", "64", "--batch_size", "16",
            "--epochs", "1", "--max_steps", "2", "--model", "LeNet"]
    out = _run(base + ["--teacher", "LeNet", "--teacher_ckpt", _teacher_ckpt(tmp_path), "--distill_k",
                       "3"], tmp_path)
    assert "Epoch: 0" in out


def test_main_dist_with_a_teacher_two_ranks(tmp_path):
    _run([f"{ROOT}/main_dist.py", "--cpu", "--nproc", "2", "--synthetic", "--synthetic_size", "64",
          "--batch_size", "16", "--epochs", "1", "--max_steps", "2", "--model", "LeNet", "--output_dir",
          str(tmp_path / "o"), "--teacher", "LeNet", "--teacher_ckpt", _teacher_ckpt(tmp_path),
          "--distill_tail", "0"], tmp_path)
    assert "Train Loss" in (tmp_path / "o" / "train.log").read_text()


@pytest.mark.parametrize("extra", [["--teacher", "LeNet"], ["--teacher_ckpt", "x"],
                                   ["--teacher", "LeNet", "--teacher_ckpt", "x", "--distill_k", "11"],
                                   ["--teacher", "LeNet", "--teacher_ckpt", "x", "--distill_temp", "0"]])
def test_bad_arguments(extra):
    import sys

    sys.path.insert(0, ROOT)
    import main

    with pytest.raises(SystemExit):
        main.main(["--cpu", "--synthetic", *extra])
