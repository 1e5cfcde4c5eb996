"""No call asks for a launch of more threads than 32 bits count: the entry points around the expert layer, over their
range of sizes, with the first step of a launch replaced by a function that only looks at the grid (no GPU needed:
nothing is launched, and no pointer is read)."""
import ctypes
import math
import random
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

LIB = Path(__file__).resolve().parents[1] / "home-seek_amd" / "libhsmoe.so"

LAUNCH = r"""
typedef struct { unsigned x, y, z; } Dim;
unsigned long long launches, most;
int __hipPushCallConfiguration(Dim grid, Dim block, unsigned long shared, void* stream) {
  const unsigned long long g[3] = {grid.x, grid.y, grid.z}, b[3] = {block.x, block.y, block.z};
  for (int i = 0; i < 3; ++i) {
    if (g[i] * b[i] > most) most = g[i] * b[i];
    if (!(g[i] * b[i])) most = ~0ull;
  }
  ++launches;
  return 1;  /* the launch ends here */
}
int hipGetLastError(void) { return 0; }
"""


def sizes(rng, top):
    """One of [1, top], by its logarithm, or close to a power of two."""
    if rng.random() < 0.5:
        return max(1, min(top, 2 ** rng.randint(0, top.bit_length()) + rng.choice((-1, 0, 0, 1))))
    return int(math.exp(rng.uniform(0.0, math.log(top))))


def calls(rng):
    """(name, arguments) without end; addresses are aligned, and never read."""
    A, B = 1 << 20, 1 << 21  # B: one of the workspaces, of as many bytes as one may want
    many = (1 << 63) - 1
    spec = lambda **kw: bytes(_spec(**kw))
    while True:
        m, d, row, stream = sizes(rng, 2 ** 31 - 1), 8 * sizes(rng, 2048), rng.randint(0, 1), rng.randint(0, 1)
        form = rng.randint(0, 3)
        s = spec(post=rng.random() < 0.5, pre=rng.random() < 0.5, row=row, stream=stream, weight=rng.randint(0, 1), form=form)
        post, pre = _pointers(s)
        yield "hsmoe_block_norm", (A, A, m, d, s, 1.0, 1e-6, A, A if pre else None, None)
        sums = rng.random() < 0.5  # of the norms' weights; without them a workgroup for each row, as far as they go
        d_gate = A if form and (sums or form > 1) else None
        yield "hsmoe_block_norm_grad", (A, A if pre else None, A, A, m, d, s, 1.0, 1e-6, A, A, A if sums and post else None, d_gate,
                                        A if sums and pre else None, B, many, None)
        vocab, cols, kinds, off = sizes(rng, 2 ** 30 - 1), sizes(rng, 2 ** 23 - 1), (rng.randint(0, 1), rng.randint(0, 1)), rng.choice((0, 0, 4))
        yield "hsmoe_embed", (A, rng.randint(0, 1), m, A + off, cols, kinds[0], vocab, cols, 1.0, kinds[1], A, None)
        yield "hsmoe_embed_grad", (A + off, cols, kinds[0], A, rng.randint(0, 1), sizes(rng, 2 ** 24 - 1), vocab, cols, 1.0,
                                   rng.randint(0, 1), A, cols, kinds[1], B, many, None)
        k = 32 * sizes(rng, 2 ** 17 - 1)
        yield "hsmoe_fp4_quant", (A, k, kinds[0], m, k, A, A, None)
        n, apart = rng.randint(1, 200), 1 << 44
        tensors = [(i + 1) * apart for i in range(n)]
        outs = [t if rng.random() < 0.5 else t + apart // 2 for t in tensors]
        counts = [sizes(rng, 2 ** 38 - 1) if rng.random() < 0.1 else sizes(rng, 2 ** 20) for _ in range(n)]
        array = lambda c, v: (c * n)(*v)
        words, kind = array(ctypes.c_int64, counts), array(ctypes.c_int32, [kinds[0]] * n)
        yield "hsmoe_grad_norm", (n, array(ctypes.c_uint64, tensors), words, kind, ctypes.c_double(2.0), A, B, many, None)
        yield "hsmoe_clip_grads", (n, array(ctypes.c_uint64, tensors), words, kind, array(ctypes.c_uint64, outs), kind,
                                   ctypes.c_double(math.inf), 1.0, A, B, many, None)
        x = rng.randint(0, 2)
        yield "hsmoe_fp4_linear", (A, x, k, A if x == 2 else None, m, k, A, A, 8 * sizes(rng, 2 ** 28 - 1), kinds[1], A, B, many, None)


class _Spec(ctypes.Structure):
    _fields_ = [("post", ctypes.c_void_p), ("pre", ctypes.c_void_p), ("gate", ctypes.c_void_p), ("row", ctypes.c_int),
                ("stream", ctypes.c_int), ("weight", ctypes.c_int), ("gate_kind", ctypes.c_int), ("form", ctypes.c_int)]


def _spec(post, pre, row, stream, weight, form):
    A = 1 << 20
    return _Spec(A if post else None, A if pre else None, A if form else None, row, stream, weight, weight, form)


def _pointers(s):
    v = _Spec.from_buffer_copy(s)
    return v.post, v.pre


def look(launch_lib, which, rounds):
    """In a process of its own, whose launches end in launch_lib."""
    seen = ctypes.CDLL(launch_lib, mode=ctypes.RTLD_GLOBAL)
    lib = ctypes.CDLL(str(LIB))
    launches, most = (ctypes.c_ulonglong.in_dll(seen, n) for n in ("launches", "most"))
    kinds = {float: ctypes.c_float, int: ctypes.c_int64}
    refused, asked, wrong = 0, 0, []
    for _, (name, args) in zip(range(rounds), calls(random.Random(11))):
        if name != which:
            continue
        before, most.value = launches.value, 0
        rc = getattr(lib, name)(*[kinds.get(type(a), lambda v: v)(a) for a in args])
        some = launches.value > before
        refused, asked = refused + (rc != 0), asked + some
        if rc not in (0, -1, -2) or some != (rc == 0) or most.value >= 2 ** 32:
            wrong.append((rc, most.value, args))
    for w in wrong[:5]:
        print("WRONG", *w)
    print(len(wrong), refused, asked)


@pytest.fixture(scope="module")
def launch_lib(tmp_path_factory):
    if shutil.which("gcc") is None:
        pytest.skip("gcc not present")
    d = tmp_path_factory.mktemp("launch")
    (d / "launch.c").write_text(LAUNCH)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-w", str(d / "launch.c"), "-o", str(d / "liblaunch.so")], check=True, timeout=60)
    return d / "liblaunch.so"


# (name, whether there are sizes that it refuses)
@pytest.mark.parametrize("name,refuses", (("hsmoe_block_norm", True), ("hsmoe_block_norm_grad", False), ("hsmoe_embed", True),
                                          ("hsmoe_embed_grad", True), ("hsmoe_fp4_quant", True), ("hsmoe_fp4_linear", True),
                                          ("hsmoe_grad_norm", False), ("hsmoe_clip_grads", False)))
def test_no_launch_has_more_threads_than_32_bits_count(launch_lib, name, refuses):
    res = subprocess.run([sys.executable, __file__, str(launch_lib), name], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stderr[-2000:]
    wrong, refused, asked = map(int, res.stdout.splitlines()[-1].split())
    assert wrong == 0, res.stdout
    assert asked > 100 and (refused > 10) == refuses


if __name__ == "__main__":
    look(sys.argv[1], sys.argv[2], 30000)
