"""Entry points where host memory has run out: a status comes back, no C++
exception (in a process of its own, whose address space is held where it is)."""
import subprocess
import sys
import textwrap


def run(body):
    code = textwrap.dedent("""
        import ctypes as C, resource
        import numpy as np
        from alpaca_amd import _lib as L
        lib = L.lib()

        def no_more_memory():
            used = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
            resource.setrlimit(resource.RLIMIT_AS, (used, resource.getrlimit(resource.RLIMIT_AS)[1]))
            # what the allocator still holds in large pieces
            malloc = C.CDLL(None).malloc
            malloc.restype, malloc.argtypes = C.c_void_p, [C.c_size_t]
            for size in (1 << 22, 1 << 20, 1 << 18, 1 << 16):
                while malloc(size):
                    pass

        def memory_again():
            hard = resource.getrlimit(resource.RLIMIT_AS)[1]
            resource.setrlimit(resource.RLIMIT_AS, (hard, hard))
    """) + textwrap.dedent(body) + "\nprint('done', flush=True)\n"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.endswith("done\n"), (r.returncode, r.stdout, r.stderr[-2000:])


def test_rotation_table():
    run("""
        table = np.zeros((3, 1 << 15, 2), np.float32)
        want = np.zeros_like(table)
        assert lib.ahip_rope_table(3, 1 << 16, 1e4, want.ctypes.data) == 0
        no_more_memory()
        rc = lib.ahip_rope_table(3, 1 << 16, 1e4, table.ctypes.data)
        memory_again()
        assert rc == 0 and (table == want).all()
    """)
