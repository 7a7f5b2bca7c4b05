"""QNT_LIB_DIR: the C ABI and the extension for torch tensors come from that folder, both as one library."""
import os
import shutil
import subprocess
import sys

import pytest

pytest.importorskip("torch")

CHECK = """
import sys
sys.path.insert(0, {pkg!r})
import quanta_b200 as qb
qb._torch_calls()
print(*sorted({{l.split()[-1] for l in open("/proc/self/maps") if "quanta_b200" in l and ".so" in l}}), sep="\\n")
"""


def test_both_libraries_come_from_one_folder(qb, tmp_path):
    names = ["libquanta_b200.so", "quanta_b200_torch.so"]
    for n in names:
        shutil.copy(qb.LIB_DIR / n, tmp_path / n)
    r = subprocess.run([sys.executable, "-c", CHECK.format(pkg=str(qb.PKG))], env=dict(os.environ, QNT_LIB_DIR=str(tmp_path)),
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    assert r.stdout.split() == [str(tmp_path.resolve() / n) for n in names]


def test_a_folder_without_the_extension(qb, tmp_path):
    shutil.copy(qb.LIB_DIR / "libquanta_b200.so", tmp_path)
    r = subprocess.run([sys.executable, "-c", CHECK.format(pkg=str(qb.PKG))], env=dict(os.environ, QNT_LIB_DIR=str(tmp_path)),
                       capture_output=True, text=True, timeout=300)
    assert r.returncode != 0 and f"{tmp_path / 'quanta_b200_torch.so'} is missing" in r.stderr
