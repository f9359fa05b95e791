"""Arguments that the decode-step operators refuse before any device is touched."""
import ctypes
import pathlib
import subprocess

import pytest
import torch

from ncmorph_b200 import _lib, build, kv_cache, ncm_model

BF = torch.bfloat16


def pool(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("args", [(pool(2, 1, 16, 64), pool(2, 1, 16, 64)), (None, None), ([1.0], [1.0])])
def test_a_cache_lives_on_a_gpu(args):
    with pytest.raises(ValueError):
        kv_cache.KVCache(*args)


def test_rows_and_logits_live_on_a_gpu():
    t = torch.zeros((4, 32))
    with pytest.raises((ValueError, TypeError)):
        ncm_model.rope_bf16(pool(2, 64), torch.zeros(2, dtype=torch.int32), t, t, 1, 64)
    with pytest.raises((ValueError, TypeError)):
        ncm_model.process_logits(torch.zeros((1, 8)))


def test_null_context_is_refused():
    lib = _lib.load()
    cache, batch, rules, n = _lib.KvCache(), _lib.KvBatch(), _lib.LogitRules(), ctypes.c_uint64()
    c, b, r = (ctypes.byref(x) for x in (cache, batch, rules))
    calls = [lib.ncm_rope_bf16(None, None, 64, None, 64, None, None, None, 1, 1, 1, 64, 64, 0, 0, None),
             lib.ncm_kv_cache_append(None, c, b, None, 64, None, 64, None),
             lib.ncm_kv_cache_gather(None, c, b, None, None, 64, None, 64, None),
             lib.ncm_tree_attention_workspace(None, c, b, 1, 1, ctypes.byref(n)),
             lib.ncm_tree_attention(None, c, b, None, 64, None, 0, 1, 1, 1.0, None, 64, None, None, 0, None),
             lib.ncm_logits_process(None, None, 2, 8, None, 2, 8, 1, 8, r, None)]
    assert calls == [_lib.NCM_EINVAL] * len(calls)


def test_struct_sizes_are_the_headers():
    """Offsets of the ctypes structs against the C layout rules (8-byte pointers)."""
    assert ctypes.sizeof(_lib.KvCache) == 4 * 8 + 4 * 4 + 8
    assert ctypes.sizeof(_lib.KvBatch) == 3 * 8 + 8 + 2 * 4 + 8
    assert ctypes.sizeof(_lib.LogitRules) == 15 * 8


def test_numbers_of_devices_stay_apart(tmp_path):
    """The attention's plan keeps its CTAs per SM by device: what another device answers
    must not change the workspace that a caller has been told."""
    csrc = pathlib.Path(_lib.__file__).parent / "csrc"
    program = tmp_path / "numbers.cu"
    program.write_text('''#include "internal.h"
int main() {
  static ncm::DeviceNumbers n;
  if (n.get(0) != 0 || n.get(63) != 0) return 1;
  n.set(0, 4);
  n.set(63, 2);
  n.set(64, 9);
  n.set(-1, 9);
  return n.get(0) == 4 && n.get(63) == 2 && n.get(1) == 0 && n.get(64) == 0 && n.get(-1) == 0 ? 0 : 2;
}
''')
    subprocess.run([build.nvcc(), "-std=c++17", f"-I{csrc}", f"-I{csrc.parents[1] / 'include'}", str(program), "-o", str(tmp_path / "numbers")],
                   check=True)
    assert subprocess.run([str(tmp_path / "numbers")]).returncode == 0
