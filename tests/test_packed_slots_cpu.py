"""Slots of the 4-bit cache that are released and taken again while other sequences decode: what the host and the table make of their lengths."""
import torch


def cache(**kw):
    from tpp_pytorch_extension_b200._C._packed_attn import Int4Cache
    return Int4Cache(**(dict(layers=1, pages=9, kv_heads=1, head_dim=64, sequences=3, columns=4, device="cpu") | kw))


def test_a_released_slot_stays_empty_while_the_others_decode():
    c = cache()
    c.add_pages([40, 40, 40])
    c.advance(torch.tensor([0, 5, 15, 22], dtype=torch.int32))
    c.release(1)
    for _ in range(4):
        c.advance()
    assert c.lengths.tolist() == [9, 0, 11]
    c.add_pages([40, 20, 40])  # the next prompt of the slot starts at place 0 and is followed by its own tokens
    c.advance(torch.tensor([0, 0, 20, 20], dtype=torch.int32))
    c.advance()
    assert c.lengths.tolist() == [10, 21, 12]


def test_a_slot_that_was_never_taken_stays_empty():
    c = cache()
    c.add_pages([10, 0, 0])
    c.advance(torch.tensor([0, 3, 3, 3], dtype=torch.int32))
    c.advance()
    assert c.lengths.tolist() == [4, 0, 0] and c.lengths.dtype == torch.int32


def test_a_table_of_the_caller_is_looked_at_as_it_is():
    """Sequences whose first pages are gone go on; one without any page does not."""
    c = cache()
    from tpp_pytorch_extension_b200._C._packed_attn import Int4Cache
    table = torch.tensor([[3, -1, -1], [-1, -1, 0], [-1, -1, -1]], dtype=torch.int32)
    own = Int4Cache.over(c.pools, table, torch.tensor([7, 70, 0], dtype=torch.int32))
    own.advance()
    assert own.lengths.tolist() == [8, 71, 0]
