"""The native extension's build."""
import os
import shutil
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_objects_older_than_a_header_are_dropped(tmp_path):
    """hipcc's objects record no headers: one that is older than any of them is
    compiled again, a newer one is kept."""
    shutil.copy(os.path.join(ROOT, "setup.py"), tmp_path)
    csrc = tmp_path / "rl_amd" / "csrc"
    objects = tmp_path / "build" / "temp.linux" / "rl_amd" / "csrc"
    shutil.copytree(os.path.join(ROOT, "rl_amd", "csrc"), csrc)
    objects.mkdir(parents=True)
    for header in csrc.glob("*.h"):
        os.utime(header, (900, 900))
    os.utime(next(csrc.glob("*.h")), (1000, 1000))
    for name, time in (("old.o", 999), ("new.o", 1001)):
        (objects / name).write_bytes(b"")
        os.utime(objects / name, (time, time))
    subprocess.run([sys.executable, "setup.py", "--name"], cwd=tmp_path, check=True, capture_output=True, timeout=300)
    assert not (objects / "old.o").exists() and (objects / "new.o").exists()
