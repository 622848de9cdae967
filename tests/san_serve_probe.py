"""Host-side probe of the decode-step entry points for the sanitizer-built library, as san_abi_probe.py is for
wc_abi.h: NULL, zero-filled, 0xFF-filled and random argument structs, then plausible ones with some extreme fields.
Device pointers are never dereferenced on the host, and without a GPU every launch fails with an error.

usage: python san_serve_probe.py <library> <wc_serve_abi.h> <iterations> <package dir>
"""

import ctypes
import random
import sys

from san_abi_probe import prototypes


def main() -> int:
    lib = ctypes.CDLL(sys.argv[1])
    lib.wc_last_error.restype = ctypes.c_char_p
    protos = prototypes(sys.argv[2])
    sys.path.insert(0, sys.argv[4])
    from wide_compiler import _serve
    fns = {name: getattr(lib, name) for _, name, _ in protos}
    assert set(fns) == set(_serve.SIGNATURES), sorted(fns)
    rng = random.Random(20261206)
    plausible = [0, 1, 2, 3, 4, 7, 8, 16, 32, 33, 64, 128, 256, 384, 512, 1024, 4096]
    extreme = [-1, -(1 << 31), (1 << 31) - 1, 1 << 32, 1 << 40, (1 << 63) - 1, -(1 << 63)]
    calls = 0
    for it in range(int(sys.argv[3])):
        for name, f in fns.items():
            res, args = _serve.SIGNATURES[name]
            f.restype, f.argtypes = res, args
            if not args:
                f()
                continue
            cls = args[0]._type_
            blocks = [None, cls(), cls.from_buffer_copy(b"\xff" * ctypes.sizeof(cls)),
                      cls.from_buffer_copy(bytes(rng.getrandbits(8) for _ in range(ctypes.sizeof(cls))))]
            for _ in range(6):
                a = cls()
                odd = rng.choice([0.0, 0.05, 0.2])
                for field, kind in a._fields_:
                    if kind is ctypes.c_void_p:
                        v = None if rng.random() < 0.1 else 0x7F0000000000 + 4096 * rng.randrange(1 << 16)
                    elif kind is ctypes.c_float:
                        v = rng.choice([0.0, 1e-6, 0.125, float("nan")])
                    elif field == "bits":
                        v = rng.choice([0, 8, 0, 8, 4])
                    elif field == "group":
                        v = rng.choice([32, 64, 128, 48])
                    elif field == "position_bytes":
                        v = rng.choice([4, 8, 4, 8, 2])
                    elif "dtype" in field:
                        v = rng.choice([0, 1, 2, 0, 1, 2, 9])
                    else:
                        v = rng.choice(extreme) if rng.random() < odd else rng.choice(plausible)
                        if kind is ctypes.c_int32:
                            v = max(min(v, (1 << 31) - 1), -(1 << 31))
                    setattr(a, field, v)
                blocks.append(a)
            for a in blocks:
                ref = None if a is None else ctypes.byref(a)
                f(ref) if len(args) == 1 else f(ref, None)
                assert isinstance(lib.wc_last_error(), bytes)
                calls += 1
    print(f"san_serve_probe: {calls} calls over {len(fns)} entry points, no sanitizer report", flush=True)
    return 0


if __name__ == "__main__":
    sys.exit(main())
