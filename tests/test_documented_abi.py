"""The library version that the repository's documents show callers is the library's."""

import re
from pathlib import Path

from parakeet_amd import _lib

ROOT = Path(__file__).resolve().parents[1]


def test_documents_name_the_library_version():
    named = [int(v) for p in sorted(ROOT.glob("*.md")) for v in re.findall(r"pk_abi_version\(\)`? ?(?:==|returns) ?(\d+)", p.read_text())]
    assert named and set(named) == {_lib.ABI_VERSION}
