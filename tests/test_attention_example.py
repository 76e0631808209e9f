"""The serving loop that the documentation shows, run with stand-ins for the layers: every kind of step
has to give the calls arguments that they take."""
import pathlib
import types

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent


@pytest.mark.parametrize("new_lens", [[5, 0, 0], [1, -1, 3], [-1, -1, -1], [0, 0, 0], [7]])
def test_documented_step(new_lens):
    text = (ROOT / "INTEGRATION.md").read_text()
    source = text[text.index("def step(new_lens, x)"):].split("\n\n")[0]
    tokens, seen = sum(max(n, 0) for n in new_lens), []

    class X:
        shape = (tokens, 64)

        def __add__(self, other):
            return self

    def layer(x, cache, i, t, max_q_len, max_kv_len):
        assert max_q_len >= 0 and max_q_len == max(0, max(new_lens)) and max_kv_len == 9 and t == "tables"
        seen.append(i)
        return x

    def cache_step(lens, max_tokens):
        assert lens == new_lens and max_tokens == tokens
        return "tables"

    names = dict(torch=types.SimpleNamespace(tensor=lambda v, dtype, device: v, int32=None), layers=[layer, layer],
                 norm=lambda x: x, longest=9, cache=types.SimpleNamespace(step=cache_step))
    exec(source, names)
    names["step"](new_lens, X())
    assert seen == [0, 1]
