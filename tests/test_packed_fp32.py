"""CPU: packed FP32 instructions (two F32 operations each) stay out of the GPU code: some of their forms have given wrong results
now and then, with no error, and they are no faster here (2.0 ns per instruction against 1.1 for one F32 operation)."""
import re

from test_tool_rules import sources

PACKED = re.compile(r"\bv_pk_(?:add|mul|fma|mov)_(?:f32|b32)\b")


def test_no_source_writes_them_by_hand():
    assert [p for p, text in sources("cyberether_amd", "integration", "oracle", "tools") if PACKED.search(text)] == []
