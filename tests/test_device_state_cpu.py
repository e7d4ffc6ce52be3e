"""What the host code of a kernel remembers between calls belongs to one GPU, and several threads may look at it."""
import os
import re

import pytest

import tnn_b200

KERNELS = os.path.join(os.path.dirname(tnn_b200.__file__), "csrc", "kernels")


@pytest.mark.parametrize("name", ["newton_schulz", "token_logprob", "embedding", "muon"])
def test_remembered_values_are_per_device_and_atomic(name):
    """These operators go to the device of their tensors, whichever is current: nothing found on one GPU is used for another."""
    text = re.sub(r"[ \t]*//.*", "", open(os.path.join(KERNELS, f"{name}.cu")).read())
    held = [line.strip() for line in re.findall(r"^[ \t]+static .*$", text, re.M) if not re.match(r"\s*static (constexpr|__device__)", line)]
    held = [line for line in held if not re.search(r"\)\s*\{?$|\) (const )?\{", line)]  # (member functions)
    assert all(re.match(r"static std::atomic<\w+> \w+\[\w+\];", line) for line in held), held
