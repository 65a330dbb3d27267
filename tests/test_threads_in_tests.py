"""CPU: a test whose threads die or stay behind does not pass."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))

DIES = """
import threading
def test_dies():
    t = threading.Thread(target=lambda: 1 / 0)
    t.start()
    t.join()
"""
STAYS = """
import threading, time
def test_stays():
    t = threading.Thread(target=time.sleep, args=(3,))
    t.start()
    t.join(0.01)
"""
ENDS = """
import threading
def test_ends():
    t = threading.Thread(target=lambda: None)
    t.start()
    t.join()
"""


@pytest.mark.parametrize("text,status,found", [(DIES, 1, "ZeroDivisionError"), (STAYS, 1, "still run"), (ENDS, 0, "1 passed")],
                         ids=["dies", "stays", "ends"])
def test_threads(tmp_path, text, status, found):
    (tmp_path / "conftest.py").write_text(open(os.path.join(HERE, "conftest.py")).read())
    (tmp_path / "test_it.py").write_text(text)
    done = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", str(tmp_path)], cwd=str(tmp_path),
                          capture_output=True, text=True, timeout=100)
    assert done.returncode == status and found in done.stdout, done.stdout + done.stderr
