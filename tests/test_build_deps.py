"""A source is compiled again when any header it includes, itself or through another, is newer than its object file."""
import os
import re

import pytest

from vearo_b200 import build as b


def included(path, seen):
    for name in re.findall(r'^\s*#include\s+"([^"]+)"', open(path).read(), flags=re.M):
        at = os.path.realpath(os.path.join(os.path.dirname(path), name))
        if os.path.exists(at) and at not in seen:
            seen.add(at)
            included(at, seen)
    return seen


@pytest.mark.parametrize("src", b.sources(), ids=os.path.basename)
def test_every_included_header_is_looked_at(src):
    looked_at = {os.path.realpath(d) for d in b._deps(src)}
    assert included(src, set()) <= looked_at
