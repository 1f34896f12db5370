"""Which files with per-head norms of queries and keys the engine opens."""
import struct

import pytest

TINY = dict(hidden_size=128, num_layers=2, num_heads=2, num_kv_heads=1, intermediate_size=64, vocab_size=64,
            max_position_embeddings=64, rope_theta=10000.0, rms_eps=1e-5, dtype=0)
KEY = b"general.architecture" + struct.pack("<IQ", 8, 5)


def error(vsl, path, **kw):
    """What opening the file fails with: "" where it opens (without a GPU it fails for want of a device)."""
    try:
        vsl.Engine(path, **kw).close()
        return ""
    except vsl.VslError as e:
        return str(e)


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("qk_norm", [True, False])
def test_norms_of_another_architecture_are_refused(vsl, tmp_path, qk_norm, halves):
    path = tmp_path / "m.gguf"
    vsl.write_synthetic_gguf(path, TINY, qk_norm=qk_norm)
    assert "architecture" not in error(vsl, path, rope_halves=halves)
    data = path.read_bytes()
    assert data.count(KEY + b"llama") == 1
    path.write_bytes(data.replace(KEY + b"llama", KEY + b"other"))
    got = error(vsl, path, rope_halves=halves)
    assert ('architecture "other"' in got) == qk_norm
