"""Pool formats at configuration time: what could never be written is refused before pools are allocated."""
import pytest

from distserve_b200.config import CacheConfig, KVModelConfig, ParallelConfig
from distserve_b200.worker import KVWorker


@pytest.mark.parametrize("block_size", [1, 6, 18])
def test_quantised_blocks_of_no_multiple_of_four_tokens(block_size):
    CacheConfig(block_size, 8)
    with pytest.raises(ValueError, match="multiple of 4 tokens"):
        CacheConfig(block_size, 8, kv_format="e4m3")


@pytest.mark.parametrize("head_dim,dtype", [(128, "float32"), (72, "float16"), (8, "bfloat16"), (272, "float16")])
def test_quantised_pools_that_no_operator_could_write(head_dim, dtype):
    model = KVModelConfig(2, 4, head_dim, dtype)
    model.check_kv_format("model")
    with pytest.raises(ValueError, match="e4m3 pools hold rows of float16 or bfloat16"):
        model.check_kv_format("e4m3")
    with pytest.raises(ValueError, match="e4m3 pools hold rows of float16 or bfloat16"):
        KVWorker(0, "decoding", model, CacheConfig(16, 8, kv_format="e4m3"))


@pytest.mark.parametrize("head_dim,dtype", [(16, "float16"), (64, "bfloat16"), (80, "float16"), (256, "bfloat16")])
def test_quantised_pools_that_can_be_written(head_dim, dtype):
    KVModelConfig(2, 4, head_dim, dtype).check_kv_format("e4m3")
