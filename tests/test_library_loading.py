"""Loading the kernel library (no GPU needed): threads whose first calls come together, and a library that does not fit its sources."""
import threading

import pytest

from carla_garage_amd import _lib


def test_first_calls_of_several_threads():
  for _ in range(5):
    lib, together, errors, got = _lib._Lib(), threading.Barrier(8), [], []

    def call():
      together.wait()
      try:
        got.append(lib.raw('tfpp_version')())
        lib.raw('tfpp_diff_attn_fwd_partial_floats')
      except Exception as e:  # noqa: BLE001
        errors.append(e)

    threads = [threading.Thread(target=call) for _ in range(8)]
    for t in threads:
      t.start()
    for t in threads:
      t.join()
    assert not errors and got == [_lib.ABI_VERSION] * 8


def test_a_library_of_other_sources_is_refused_every_time(monkeypatch):
  lib = _lib._Lib()
  monkeypatch.delenv('TFPP_SKIP_HASH_CHECK', raising=False)
  monkeypatch.setattr(_lib, 'source_hash', lambda: 1)
  for _ in range(2):
    with pytest.raises(_lib.TfppError, match='other sources'):
      lib.load()
  monkeypatch.undo()
  assert lib.load() is lib
