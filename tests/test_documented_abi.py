"""The library version that the repository's documents show callers is the library's."""

import re
from pathlib import Path

from parakeet_amd import _lib

ROOT = Path(__file__).resolve().parents[1]


def test_documents_name_the_library_version():
    guides = [t for t in (p.read_text() for p in sorted(ROOT.glob("*.md"))) if 'ctypes.CDLL("libparakeet_paged.so")' in t]
    named = [int(v) for t in guides for v in re.findall(r"pk_abi_version\(\)`? ?(?:==|returns) ?(\d+)", t)]
    assert named and set(named) == {_lib.ABI_VERSION}
