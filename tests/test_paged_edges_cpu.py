"""What of the paged cache's edges needs no GPU."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def in_a_process_of_its_own(code):
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout + r.stderr


def test_first_calls_of_several_threads_load_the_operators_once():
    in_a_process_of_its_own("""
import threading
import ads_model_kernel_library_b200.gdpa as G
paged = G.paged
paged._operators = None  # as on an import that could not load them
made, meet, errors = [], threading.Barrier(8), []
init = paged._Operators.__init__
def counted(self):
    made.append(self)
    threading.Event().wait(0.05)
    init(self)
paged._Operators.__init__ = counted
def first():
    meet.wait()
    try:
        assert paged._operators or paged._load()
    except Exception as e:
        errors.append(e)
threads = [threading.Thread(target=first) for _ in range(8)]
[t.start() for t in threads], [t.join() for t in threads]
assert not errors and len(made) == 1, (errors, len(made))
print("ok")
""")
