"""What no source file of this repository may hold."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SUFFIXES = (".py", ".hip", ".hpp", ".h", ".inc", ".cpp", ".s", ".sh", ".map", ".cfg", ".ini", ".toml", ".txt", ".cmake")
FOLDERS = ("bluenoise", "bndm_amd", "include", "oracle", "perf", "scripts", "tests", "tools")


def sources():
    for top, names in [(ROOT, os.listdir(ROOT))] + [(top, names) for f in FOLDERS for top, _, names in os.walk(os.path.join(ROOT, f))]:
        for name in names:
            path = os.path.join(top, name)
            if (name.endswith(SUFFIXES) or name == "Makefile") and os.path.isfile(path):
                yield path


def test_no_source_writes_through_the_scalar_data_cache():
    """Kernels write through vector stores alone: the scalar cache's stores, atomics, write-back and discard have no place in them, nor a name in the
    simulator's table of instructions."""
    names = re.compile(r"\bs_(?:dcache_(?:wb|discard)|(?:buffer_|scratch_)?(?:store_dword|atomic_))")
    paths = list(sources())
    assert len(paths) > 80
    found = [os.path.relpath(p, ROOT) for p in paths if names.search(open(p, encoding="utf-8", errors="replace").read())]
    assert found == []
