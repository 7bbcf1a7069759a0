"""Every kernel here writes memory through vector stores and vector atomics.

The scalar data cache is not kept coherent with the vector path, so a store, an atomic, a write-back or a discard
through it is used nowhere: not in a kernel, a microbenchmark or a build script, and not in a comment of one, where it
would be taken up again.  The search reads text only; no such instruction is assembled or run.
"""
import os
import re

import pytest

from conftest import ROOT

FOLDERS = ("include", "oracle", "perf", "profiles", "rcppsparse_amd", "tests", "tools")
SUFFIXES = (".hip", ".h", ".hpp", ".inc", ".c", ".cc", ".cpp", ".s", ".S", ".ll", ".py", ".sh", ".R", ".mk", ".cmake")
BUILD_FILES = ("Makefile", "Makevars", "Makevars.in", "CMakeLists.txt", "configure")

# The mnemonics (s_..., any width) and the compiler's builtins and intrinsics for them, whose prefix ends in _ or a dot.
WRITES = re.compile(r"(?<![a-z0-9])s[._](?:(?:scratch|buffer)[._])?(?:(?:store|atomic)[._]|dcache[._](?:wb|discard))",
                    re.IGNORECASE)


def sources():
    for name in sorted(os.listdir(ROOT)):
        if name.endswith(SUFFIXES) or name in BUILD_FILES:
            yield os.path.join(ROOT, name)
    for folder in FOLDERS:
        for where, _, names in os.walk(os.path.join(ROOT, folder)):
            for name in sorted(names):
                if name.endswith(SUFFIXES) or name in BUILD_FILES:
                    yield os.path.join(where, name)


def test_no_source_writes_through_the_scalar_cache():
    found, read = [], []
    for path in sources():
        read.append(os.path.relpath(path, ROOT))
        with open(path, encoding="utf-8", errors="replace") as f:
            found += [f"{read[-1]}:{k}: {line.strip()}" for k, line in enumerate(f, 1) if WRITES.search(line)]
    for kernel in ("colsums_kernels.hip", "rowsums.hip", "crossprod.hip"):     # the search reached the kernels
        assert any(name.endswith(kernel) for name in read), kernel
    assert not found, "\n".join(found)


# Put together from parts, so that this file passes its own search.
@pytest.mark.parametrize("prefix", ["s_", "__builtin_amdgcn_s_", "llvm.amdgcn.s."])
@pytest.mark.parametrize("parts", [("store", "dword"), ("buffer", "store", "dwordx4"), ("scratch", "store", "dword"),
                                   ("atomic", "add"), ("buffer", "atomic", "cmpswap", "x2"),
                                   ("dcache", "wb"), ("dcache", "wb", "vol"), ("dcache", "discard", "x2")])
def test_the_search_knows_the_forms(prefix, parts):
    assert WRITES.search("\t" + prefix + prefix[-1].join(parts) + " ...")


@pytest.mark.parametrize("line", ["s_load_dwordx4 s[0:3], s[4:5], 0x0", "global_atomic_add v0, v1, s[0:1]",
                                  "buffer_store_dwordx2 v[0:1], off, s[0:3], 0", "ds_store_b64 v0, v[2:3]",
                                  "__builtin_amdgcn_ds_atomic_fadd_f64(p, v)", "threads_stores_ms", "s_dcache_inv"])
def test_the_search_leaves_the_vector_path_alone(line):
    assert not WRITES.search(line)
