"""What the training step and the losses over rows of class scores refuse or survive, without a GPU."""
from __future__ import annotations

import pytest
import torch

from opencl_tf import errors


def test_targets_of_another_form_than_the_captured():
    """A captured step's buffers take what has their form; anything else is refused and leaves them as they were."""
    from opencl_tf import train
    ids, y = torch.arange(12).view(4, 3), torch.randn(4, 3)
    buffers = (torch.zeros_like(ids), torch.zeros_like(y))
    train._copy(train._copies(buffers, (ids, y), "targets"))
    assert torch.equal(buffers[0], ids) and torch.equal(buffers[1], y)
    for bad in ((ids + 1,), ids + 1, y + 1, (y, ids), (ids + 1, y[:1]), (ids[:2], y[:2]), (ids + 1, y, y), (ids + 1, y.half()),
                (ids.int(), y), [ids + 1, y], (ids + 1, None), None, ()):
        with pytest.raises(errors.InvalidArgumentError, match="captured with targets"):
            train._copy(train._copies(buffers, bad, "targets"))
        assert torch.equal(buffers[0], ids) and torch.equal(buffers[1], y)
    one = torch.zeros(4, 3)
    for good in (y, y.double(), torch.ones(4, 3, dtype=torch.uint8), y.t().contiguous().t()):  # converted, as ever
        train._copy(train._copies(one, good, "input"))
        assert torch.equal(one, good.float())
    for bad in (y[:1], y[0], y[None], y[:, :1], torch.tensor(1.0), (y,), [y], None):
        with pytest.raises(errors.InvalidArgumentError, match="captured with input"):
            train._copy(train._copies(one, bad, "input"))
    with pytest.raises(errors.InvalidArgumentError):
        train._copy(train._copies(buffers[0], y, "input"))  # would drop fractions


def test_misaligned_row_stats_are_refused():
    """Statistics are stored as pairs of floats: an address that is no multiple of 8 is refused before any launch."""
    import ctypes

    from opencl_tf import _library as L
    lib, x = L._lib, ctypes.byref(L.Logits(data=64, dtype=0, outer=1, inner=4, classes=10, outer_stride=0, inner_stride=10))
    P, odd = ctypes.c_void_p(64), ctypes.c_void_p(68)  # never looked at
    for name, args in (("token_log_probs", (P, 8, P, odd)), ("token_log_probs_grad", (P, 8, odd, P, P)),
                       ("distillation_loss", (P, 8, P, 0, 4, None, 0, 1.0, P, odd, None, None)),
                       ("distillation_loss_grad", (P, 8, P, 0, 4, None, 0, 1.0, odd, P, P))):
        assert getattr(lib, "b2_" + name)(None, x, *args) == 1
        assert L._lib.b2_last_error().decode() == name + ": row_stats must be 8-byte aligned"


def test_the_package_without_the_losses_binding():
    """Where the compiled autograd nodes cannot be loaded, the ops, layers and optimizer are there all the same, and a
    loss says what is missing."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import sys
sys.modules["opencl_tf._class_scores"] = None  # importing it fails
import torch, opencl_tf
assert callable(opencl_tf.conv2d) and callable(opencl_tf.step_ops.opencl_mse_loss) and opencl_tf.optimizers.Adam
try:
    opencl_tf.losses.token_log_probs(torch.zeros(2, 3), torch.zeros(2, dtype=torch.long))
except ImportError as e:
    assert "build.py" in str(e)
    print("refused")
"""
    package = Path(__file__).resolve().parent.parent / "opencl-tensorflow_b200"
    done = subprocess.run([sys.executable, "-c", code], cwd=package, capture_output=True, text=True, timeout=300)
    assert done.stdout.strip() == "refused", done.stderr[-2000:]


def test_the_losses_binding_is_built_again_for_another_torch(monkeypatch, tmp_path):
    """Its build depends on the installed torch and Python and on the command, not on file times alone; a build that
    fails leaves the last one as it was."""
    import importlib.util
    import types
    from pathlib import Path
    spec = importlib.util.spec_from_file_location(
        "binding_build", Path(__file__).resolve().parent.parent / "opencl-tensorflow_b200" / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    monkeypatch.setattr(build, "PKG", tmp_path)
    monkeypatch.setattr(build, "OBJ", tmp_path / "_build")
    monkeypatch.setattr(build, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    (tmp_path / "_build").mkdir()
    (tmp_path / "opencl_tf").mkdir()
    src = tmp_path / "nodes.cpp"
    src.write_text("")
    runs, status = [], 0

    def compiler(cmd, **_):
        runs.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_text(f"build {len(runs)}")
        return types.SimpleNamespace(returncode=status, stdout="", stderr="no")

    monkeypatch.setattr(build.subprocess, "run", compiler)
    out = build._compile_binding(src, False)
    assert out == tmp_path / "opencl_tf" / "_nodes.so" and out.read_text() == "build 1"
    build._compile_binding(src, False)
    assert len(runs) == 1
    with monkeypatch.context() as other:
        other.setattr(torch, "__version__", "0.0.1")
        build._compile_binding(src, False)
        assert len(runs) == 2 and out.read_text() == "build 2"
    build._compile_binding(src, False)
    assert len(runs) == 3
    build._compile_binding(src, True)
    assert len(runs) == 4 and out.read_text() == "build 4"
    status = 1
    with pytest.raises(RuntimeError, match="g\\+\\+ failed"):
        build._compile_binding(src, True)
    assert out.read_text() == "build 4" and [p.name for p in (tmp_path / "opencl_tf").iterdir()] == ["_nodes.so"]
    status = 0
    build._compile_binding(src, False)
    assert len(runs) == 5


def test_a_binding_that_does_not_compile_leaves_the_library_built(monkeypatch, tmp_path):
    import importlib.util
    import types
    from pathlib import Path
    spec = importlib.util.spec_from_file_location(
        "binding_build", Path(__file__).resolve().parent.parent / "opencl-tensorflow_b200" / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    for name in ("OBJ", "CSRC", "BINDING"):
        (tmp_path / name).mkdir()
        monkeypatch.setattr(build, name, tmp_path / name)
    monkeypatch.setattr(build, "LIB", tmp_path / "libb2ocl.so")
    monkeypatch.setattr(build, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    (tmp_path / "CSRC" / "a.cu").write_text("")
    (tmp_path / "BINDING" / "nodes.cpp").write_text("")

    def compiler(cmd, **_):
        if "nodes.cpp" in " ".join(cmd):
            return types.SimpleNamespace(returncode=1, stdout="", stderr="no header")
        Path(cmd[cmd.index("-o") + 1]).write_text("built")
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(build.subprocess, "run", compiler)
    with pytest.raises(RuntimeError, match="no header"):
        build.build()
    assert (tmp_path / "libb2ocl.so").read_text() == "built"


def test_a_captured_steps_buffers_stay_out_of_autograd():
    """Targets that a recorded network computed (a teacher's logits) are values: the buffers keep no graph of them, which
    would grow from step to step."""
    from opencl_tf import train
    teacher = torch.nn.Linear(3, 5)
    buffers = (torch.zeros(4, 5), torch.zeros(4, 5))
    for _ in range(2):
        train._copy(train._copies(buffers, (teacher(torch.randn(4, 3)), torch.randn(4, 5)), "targets"))
        assert not any(b.requires_grad for b in buffers)
