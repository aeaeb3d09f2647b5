"""What the device code of this tree must not hold, checked on its text and on what the compiler makes of it (no GPU)."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# A device program writes through vector stores and atomics only: scalar memory stores and atomics and the scalar data
# cache's write-back and discard are refused on the machines this library runs on, in comments and patches too, and one
# file that names them keeps the whole tree from being run there.
SCALAR_CACHE_WRITES = re.compile(r"\bs_(?:(?:buffer_|scratch_)?(?:store_(?:dword|b\d)|atomic_)|dcache_(?:wb|discard))", re.I)
PROGRAM_TEXT = (".hip", ".cpp", ".hpp", ".c", ".h", ".s", ".py", ".sh", ".patch", ".diff", ".cmake", ".mk")
NOT_SOURCE = {"build", "lib", "_work", "gpurun_out", "__pycache__"}      # built files and scratch folders, none of them tracked


def program_files():
    for folder, subs, names in os.walk(ROOT):
        subs[:] = sorted(s for s in subs if s not in NOT_SOURCE and not s.startswith("."))
        for n in sorted(names):
            if n.endswith(PROGRAM_TEXT) or n == "Makefile":
                yield os.path.join(folder, n)


def test_the_pattern_knows_the_instructions():
    for name in ("s_" + "atomic_add", "s_" + "buffer_atomic_swap_x2", "s_" + "store_dwordx2", "s_" + "buffer_store_dword",
                 "s_" + "scratch_store_dwordx4", "s_" + "store_b64", "s_" + "dcache_wb_vol", "s_" + "dcache_discard_x2"):
        assert SCALAR_CACHE_WRITES.search('asm volatile("' + name + ' %0");'), name
    for name in ("s_load_dword", "s_buffer_load_dwordx4", "s_waitcnt", "s_store", "no_stores_elsewhere", "s_dcache_inv"):
        assert not SCALAR_CACHE_WRITES.search(name), name


def test_no_program_text_names_a_write_through_the_scalar_cache():
    found = []
    for path in program_files():
        with open(path, encoding="utf-8", errors="replace") as f:
            for no, line in enumerate(f, 1):
                if SCALAR_CACHE_WRITES.search(line):
                    found.append(f"{os.path.relpath(path, ROOT)}:{no}")
    assert not found, found
