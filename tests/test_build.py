"""The Makefile's rules, without building anything (make -n prints what it would run)."""
import os
import subprocess

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lp-gnn_amd")


def _would_run(tmp_path, version):
    """make's plan for a host module built a moment ago, beside a torch of this version."""
    torch = tmp_path / "torch"
    torch.mkdir(exist_ok=True)
    (torch / "version.py").write_text(f"__version__ = {version!r}\n")
    os.utime(torch / "version.py", (1, 1))  # (an installer may keep the archive's old times)
    obj, host = tmp_path / "obj", tmp_path / "_host.so"
    p = subprocess.run(["make", "-C", LIB, f"TORCH={torch}", f"OBJDIR={obj}", f"HOST={host}", "-n", str(host)],
                       capture_output=True, text=True, check=True)
    return p.stdout


def test_host_module_is_built_again_for_another_torch(tmp_path):
    """It is compiled against the installed torch, newer or older than the last one."""
    host = tmp_path / "_host.so"
    for version in ("2.10.0", "2.11.0", "2.10.0"):
        assert "g++" in _would_run(tmp_path, version)
        stamp = [w for w in _would_run(tmp_path, version).split() if os.path.basename(w).startswith("torch-")]
        assert stamp
        subprocess.run(["make", "-s", "-C", LIB, f"TORCH={tmp_path / 'torch'}", f"OBJDIR={tmp_path / 'obj'}", stamp[-1]],
                       check=True)
        host.write_text("")
        assert "g++" not in _would_run(tmp_path, version)
