"""Status texts say what the grouped and MXFP4 calls may have met."""
from gemm_b200 import _lib


def test_texts_name_the_causes_of_the_grouped_and_mxfp4_calls():
    recorded = _lib.status_str(5)
    assert "offsets" in recorded and "wait" in recorded and "neogemm_device_status" in recorded
    unsupported = _lib.status_str(2)
    assert "1024 groups" in unsupported and "MXFP4" in unsupported and "multiples of 8" in unsupported
    assert "offsets" in str(_lib.NeoGemmError(5, recorded))
