"""CPU test of the binding: a cache in 8 bits has two fields more, and a struct without them is refused before the library reads past it."""
import pytest

import es_hip_quant as E

CALLS = {
    "kv_append_dev": (1, None, 1, E.F32, 4096, 0, 4096, 0),
    "attn_decode_workspace": (1, 4),
    "attn_prompt_workspace": (1, 9, 4, E.F32),
    "attn_workspace_upto": (1, 9, 4),
    "attn_decode_dev": (1, 4, E.F32, 4096, 0, 0.1, 0, 4096, 0, 4096, 1 << 30),
    "attn_prompt_dev": (1, 4096, 9, 4, E.F32, 4096, 0, 0.1, 0, 4096, 0, 4096, 1 << 30),
    "attn_decode_sinks_dev": (1, 4, E.F32, 4096, 0, 0.1, 5, 1, 4096, 0, 4096, 1 << 30),
    "attn_prompt_sinks_dev": (1, 4096, 9, 4, E.F32, 4096, 0, 0.1, 5, 1, 4096, 0, 4096, 1 << 30),
    "kv_copy_pages_dev": (1, 0, [1], [2]),
}
FIELDS = (4, 128, 16, 100, 4096, 8192, 4096, 4096, None, 8, 64)


@pytest.mark.parametrize("name", CALLS)
def test_an_8_bit_cache_without_its_scales(hiplib, name):
    with pytest.raises(ValueError, match="Kv8"):
        getattr(hiplib, name)(E.Kv(E.F8, *FIELDS), *CALLS[name])


def test_others_pass(hiplib):
    for kv in (E.Kv(E.F16, *FIELDS), E.Kv8(E.F16, *FIELDS, None, None), E.Kv8(E.F8, *FIELDS, 4096, 4096)):
        assert hiplib.attn_workspace_upto(kv, 1, 9, 4) > 0
