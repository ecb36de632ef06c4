"""The grids of calls of the C ABI, without a GPU: loads libsbq.so over the
launch recorder (launch_trace.cpp) and runs calls on made-up device addresses,
which host code never reads.

    grids.py RECORDER LIBRARY PACKAGE < calls > grids

stdin: a JSON list of calls [entry point, argument, ...], an argument "@i" the
address (i + 1) << 40; stdout: for each, {"rc": status, "launches": [[grid xyz,
block xyz], ...]}.  A process of its own, as dispatch.py."""
import ctypes
import json
import sys


def main():
    rec = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
    L = ctypes.CDLL(sys.argv[2])
    sys.path.insert(0, sys.argv[3])
    from _lib import SIGNATURES

    out = []
    buf, dims = ctypes.create_string_buffer(4096), (ctypes.c_int64 * 7)()
    for name, *args in json.load(sys.stdin):
        f = getattr(L, name)
        f.restype, f.argtypes = SIGNATURES[name]
        rec.trace_reset()
        rc = f(*[(int(a[1:]) + 1) << 40 if isinstance(a, str) else a for a in args])
        launches = []
        for i in range(rec.trace_count()):
            rec.trace_get(i, buf, ctypes.c_size_t(len(buf)), dims)
            launches.append([list(dims)[0:3], list(dims)[3:6]])
        out.append({"rc": rc, "launches": launches})
    json.dump(out, sys.stdout)


if __name__ == "__main__":
    main()
