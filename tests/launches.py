"""Which kernels the library's entry points launch, without a GPU: `launched(code)`
runs `code` in a child process whose HIP runtime is tests/cpp/launches.cpp, with `L`
the library, `shown()` the launches since the last look as (kernel, grid x, grid y,
block) and `A(i)` addresses far from one another; `out`, which the code sets, comes
back."""
import json
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_RECORDER = os.path.join(ROOT, "tests", "cpp", "_build", "liblaunches.so")

_CHILD = """
import ctypes, json, sys
sys.path.insert(0, {root!r})
R = ctypes.CDLL({recorder!r}, ctypes.RTLD_GLOBAL)  # before the library, so that it is found first
R.launches_lines.restype = ctypes.c_char_p
from ark_amd import _abi, _lib
L = _lib.lib()
A = lambda i: i << 44

def shown():
    text = R.launches_lines().decode()
    R.launches_clear()
    rows = [line.split(" ", 3) for line in text.splitlines()]
    return [(name, int(x), int(y), int(b)) for x, y, b, name in rows]

def ok(rc):
    assert rc == 0, L.ark_opt_last_error().decode()

{code}
print(json.dumps(out))
"""


def launched(code):
    subprocess.run(["make", "-C", os.path.join(ROOT, "tests", "cpp"), "_build/liblaunches.so"],
                   check=True, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    r = subprocess.run([sys.executable, "-c", _CHILD.format(root=ROOT, recorder=_RECORDER, code=code)],
                       stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    return json.loads(r.stdout.splitlines()[-1])
