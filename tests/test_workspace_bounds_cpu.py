"""Workspaces that are sized once for the longest sequence have to do for every shorter one."""
import pytest

torch = pytest.importorskip("torch")


def chunks(rows, n, sms):
    """How the order-free P.V kernel cuts n tokens of `rows` (batch, KV head) rows: about eight parts per SM, of whole 128 tokens, at least 256."""
    want = -(-sms * 8 // rows)
    size = max(256, -(-(-(-n // want)) // 128) * 128)
    return -(-n // size)


@pytest.mark.parametrize("rows", [1, 3, 8, 32, 75, 150, 256, 512, 2048])
def test_shorter_sequences_have_room(akv_lib, rows):
    sms = torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 148
    last_v = last_step = 0
    for n in sorted(set(range(64, 30000, 64 * 37)) | {4096, 4160, 10240, 10304, 12288, 12352, 24576, 24640}):
        v = akv_lib.akv_v_cache_compute_scratch_bytes(rows, 1, 4, n)
        step = akv_lib.akv_decode_scratch_bytes_ex(rows, 1, 4, 128, n, 2)
        assert v >= last_v and step >= last_step, n
        assert v >= rows * 4 * max(chunks(rows, m, sms) for m in range(64, n + 1, 64)) * 128 * 4, n
        last_v, last_step = v, step
