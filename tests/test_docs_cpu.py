"""What the documents name has to be there."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("doc", ["DESIGN.md", "INTEGRATION.md", "README.md", "profiles/INDEX.md"])
def test_every_tool_that_a_document_names_exists(doc):
    with open(os.path.join(ROOT, doc)) as f:
        named = sorted(set(re.findall(r"tools/[\w./]+\.\w+", f.read())))
    assert [t for t in named if not os.path.exists(os.path.join(ROOT, t))] == []
