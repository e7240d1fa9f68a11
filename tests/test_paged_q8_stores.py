"""What a cache in 8 bits reads and writes past the caches: whole lines."""
import re

from test_product_distances import _assembly, _kernels


def test_reading_back_writes_whole_lines(tmp_path):
    """A store past the caches is written as it is: the threads of a wavefront write 16 bytes beside one another, one store of keys and one of values each (two stores of a thread
    that lie side by side leave holes in each other's lines)."""
    seen = 0
    for name, code, _ in _kernels(_assembly("paged_q8_append", tmp_path)):
        if "paged_read_q8" in name:
            stores = [(op, operands) for op, operands, _ in code if op.startswith(("global_store", "flat_store", "buffer_store"))]
            assert len(stores) == 2 and all(op == "global_store_dwordx4" and operands[-1].split()[-1] == "nt" for op, operands in stores), (name, stores)
            seen += 1
    assert seen == 4


def test_appending_reads_whole_lines_past_the_caches(tmp_path):
    """A load takes half of each of several heads; of half a line at a time each comes twice."""
    past = []
    for name, code, _ in _kernels(_assembly("paged_q8_append", tmp_path)):
        m = re.search(r"paged_append_q8_kernelI(DF16b|f)Li(\d+)ELi\d+E", name)
        if m and any(op.startswith("global_load") and operands[-1].split()[-1] == "nt" for op, operands, _ in code):
            past.append(name)
            assert int(m[2]) // 2 * (4 if m[1] == "f" else 2) >= 128, name
    assert len(past) == 24   # three sizes of head and type, four of blocks, rotated or not
