"""What the host code of libblp.so launches, without a GPU: calls of its C entry points in a child process in which hip_stub.c stands
in for the runtime's launch calls.

    run([("blp_lookup", [...], None), ...]) -> [{"rc", "error", "launches": [{"name", "grid", "block", "product"}]}]

The third item of a call is None, or (i, e): its launch number i fails with the runtime's error e. Arguments: numbers, and None
for null pointers. Pointers are not read by the host code.
"""
import ctypes
import json
import os
import re
import struct
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))


def run(calls):
    with tempfile.TemporaryDirectory() as tmp:
        stub = os.path.join(tmp, "hip_stub.so")
        subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-Wall", "-o", stub, os.path.join(HERE, "hip_stub.c")], check=True)
        r = subprocess.run([sys.executable, os.path.abspath(__file__), stub], input=json.dumps(calls), capture_output=True, text=True,
                           timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    return json.loads(r.stdout)


def _product(name, raw):
    """k_product<T, LP, LQ, SEGS, ...>'s template arguments and the Problem it was given."""
    args = re.search(r"k_productILi(\d)ELi(\d)ELi(\d)ELi(\d)E", name)
    if not args:
        return None
    t, lp, lq, segs = (int(x) for x in args.groups())
    k, slice_, tiles_p, tiles_q = struct.unpack_from("<qiii", raw, 48)
    return {"type": t, "lp": lp, "lq": lq, "segments": segs, "k": k, "slice": slice_, "tiles_p": tiles_p, "tiles_q": tiles_q,
            "p_rows": struct.unpack_from("<q", raw, 16)[0], "q_rows": struct.unpack_from("<q", raw, 40)[0]}


def _child(stub):
    S = ctypes.CDLL(stub, mode=ctypes.RTLD_GLOBAL)
    S.stub_name.restype = ctypes.c_char_p
    S.stub_first.restype = ctypes.POINTER(ctypes.c_ubyte)
    sys.path.insert(0, os.path.join(os.path.dirname(HERE), "bipartite-link-prediction_amd"))
    from blp import _lib, latent  # noqa: F401  (registers its entry points)

    L, out = _lib.lib(), []
    for fn, args, fail in json.load(sys.stdin):
        S.stub_reset(*(fail or (-1, 0)))
        rc = getattr(L, fn)(*args)
        launches = []
        for i in range(S.stub_count()):
            shape = (ctypes.c_uint32 * 6)()
            S.stub_shape(i, shape)
            name = S.stub_name(i).decode()
            launches.append({"name": name, "grid": list(shape[:3]), "block": list(shape[3:]),
                             "product": _product(name, bytes(S.stub_first(i)[:88]))})
        out.append({"rc": rc, "error": L.blp_last_error().decode() if rc else "", "launches": launches})
    json.dump(out, sys.stdout)


if __name__ == "__main__":
    _child(sys.argv[1])
