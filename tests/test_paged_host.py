"""CPU: what the bindings of the paged cache refuse before anything is launched."""
import pytest
import torch

from pet_b200 import lib as L
from pet_b200 import ops


class _NoCalls:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


@pytest.fixture
def ctx():
    c = ops.Context.__new__(ops.Context)
    c.lib, c.h, c._plans, c.device = _NoCalls(), None, {}, torch.device("cpu")
    c._kv_device, c._kv_need = -1, {}  # (what tensors on the host answer)
    return c


def args(tokens=2, seqs=2, heads=2, q_heads=4, dim=64, dtype=torch.bfloat16):
    return dict(q=torch.zeros(tokens, q_heads, dim, dtype=dtype), k_cache=torch.zeros(3, 16, heads, dim, dtype=dtype), v_cache=torch.zeros(3, 16, heads, dim, dtype=dtype),
                page_table=torch.zeros(seqs, 2, dtype=torch.int32), kv_lens=torch.ones(seqs, dtype=torch.int32))


BAD = [("q", torch.zeros(2, 4, 64)), ("q", torch.zeros(2, 4, 32, dtype=torch.bfloat16)), ("q", torch.zeros(2, 256, dtype=torch.bfloat16)),
       ("v_cache", torch.zeros(3, 16, 2, 64)), ("v_cache", torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)), ("k_cache", torch.zeros(3, 32, 64, dtype=torch.bfloat16)),
       ("page_table", torch.zeros(2, 2, dtype=torch.int64)), ("page_table", torch.zeros(3, 2, dtype=torch.int32)), ("page_table", torch.zeros(2, dtype=torch.int32)),
       ("kv_lens", torch.ones(2)), ("kv_lens", torch.ones(2, 1, dtype=torch.int32)), ("q_starts", torch.zeros(2, dtype=torch.int32)),
       ("q_starts", torch.zeros(3, dtype=torch.int64)), ("out", torch.zeros(2, 4, 64)), ("out", torch.zeros(3, 4, 64, dtype=torch.bfloat16))]


@pytest.mark.parametrize("name,value", BAD)
def test_attention_refuses(ctx, name, value):
    a = args()
    a[name] = value
    with pytest.raises(L.PetError) as e:
        ctx.attention_paged(**a)
    assert e.value.status == L.ERR_INVALID
    with pytest.raises(L.PetError):
        ctx.attention_prefix(prefix_table=torch.zeros(1, dtype=torch.int32), prefix_len=3, **a)


@pytest.mark.parametrize("length", [-1, 17])
def test_prefix_refuses_lengths_its_table_does_not_hold(ctx, length):
    with pytest.raises(L.PetError) as e:
        ctx.attention_prefix(prefix_table=torch.zeros(1, dtype=torch.int32), prefix_len=length, **args())
    assert e.value.status == L.ERR_INVALID


def test_values_of_a_head_must_be_contiguous(ctx):
    a = args()
    a["k_cache"] = torch.zeros(3, 16, 64, 2, dtype=torch.bfloat16).transpose(2, 3)
    with pytest.raises(L.PetError) as e:
        ctx.attention_paged(**a)
    assert e.value.status == L.ERR_UNSUPPORTED
    a = args()
    with pytest.raises(L.PetError) as e:
        ctx.attention_paged(out=torch.zeros(2, 64, 4, dtype=torch.bfloat16).transpose(1, 2), **a)
    assert e.value.status == L.ERR_UNSUPPORTED


@pytest.mark.parametrize("change", [dict(k=torch.zeros(2, 2, 64, dtype=torch.float16)), dict(v=torch.zeros(1, 2, 64, dtype=torch.bfloat16)),
                                    dict(v=torch.zeros(2, 2, 64)), dict(k=torch.zeros(2, 3, 64, dtype=torch.bfloat16)), dict(q=torch.zeros(2, 4, 64)),
                                    dict(q_out=torch.zeros(2, 4, 64, dtype=torch.bfloat16)), dict(inv_freq=torch.ones(32, dtype=torch.float64)),
                                    dict(inv_freq=torch.ones(2, 32))])
def test_append_refuses(ctx, change):
    a = args()
    a.pop("q")
    a.update(k=torch.zeros(2, 2, 64, dtype=torch.bfloat16), v=torch.zeros(2, 2, 64, dtype=torch.bfloat16))
    a.update(change)
    with pytest.raises(L.PetError) as e:
        ctx.kv_append(**a)
    assert e.value.status == L.ERR_INVALID


def test_entry_points_without_a_context():
    lib = L.load()
    cache, seqs, rows = bytes(L.KV_CACHE.size), bytes(L.KV_SEQS.size), bytes(L.KV_ROWS.size)
    assert lib.petb200_kv_append_run(None, cache, seqs, rows, rows, rows, rows, 0, 0, None, 0, 0, 0, None) == L.ERR_INVALID
    assert lib.petb200_attention_paged_run(None, cache, seqs, rows, rows, 1, 1, 1.0, None, 0, None) == L.ERR_INVALID
    assert lib.petb200_attention_prefix_run(None, cache, seqs, None, 0, rows, rows, 1, 1, 1.0, None, 0, None) == L.ERR_INVALID


def test_descriptors_are_packed_as_the_header_lays_them_out(tmp_path):
    """Sizes and offsets of the C structures, asked of the compiler."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"petb200_kv_cache": (L.KV_CACHE, "k v k_page k_slot k_head v_page v_slot v_head dtype pages page_size heads dim"),
             "petb200_kv_seqs": (L.KV_SEQS, "page_table kv_lens q_starts table_stride table_width seqs tokens"), "petb200_kv_rows": (L.KV_ROWS, "p tok head")}
    lines = ['#include "petb200.h"', "#include <cstdio>", "#include <cstddef>", "int main() {"]
    for n, (_, fields) in names.items():
        lines.append(f'printf("%zu", sizeof({n}));')
        lines += [f'printf(" %zu", offsetof({n}, {f}));' for f in fields.split()]
        lines.append('printf("\\n");')
    src, exe = tmp_path / "o.cc", tmp_path / "o"
    src.write_text("\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["g++", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    for line, (packed, fields) in zip(out, names.values()):
        size, *offsets = map(int, line.split())
        assert size == packed.size
        values = list(range(1, 1 + len(offsets)))
        blob = packed.pack(*values)
        for v, o in zip(values, offsets):
            assert blob[o] == v and blob[o + 1] == 0


@pytest.mark.parametrize("pos0", [2 ** 31, -2 ** 31 - 1, 2 ** 40])
def test_append_refuses_positions_past_32_bits(ctx, pos0):
    """They would reach the library cut to 32 bits, and turn the keys by other angles."""
    a = args()
    q = a.pop("q")
    with pytest.raises(L.PetError) as e:
        ctx.kv_append(k=q[:, :2], v=q[:, 2:], inv_freq=torch.ones(32), pos0=pos0, **a)
    assert e.value.status == L.ERR_INVALID
