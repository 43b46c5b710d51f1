// What packed attention's copies of keys and values to LDS ask for, apart from
// the kernel (packed.hip) so that a host program checks every lane's reads.
//
// A step's rows are copied 16 bytes a lane by buffer loads from the step's first
// row on, whose reads past the buffer's bytes the hardware drops and gives zeros
// for. It compares an address's vector offset with those bytes, and no scalar
// one: where a read lies is all in the vector offset. Offsets stay in 32 bits for
// rows of less than 2^25 bytes apart and steps of up to 128 of them.
#pragma once

namespace mi::packed_copies
{
  constexpr int pieces(int hd) { return hd / 8; } // of 16 bytes, a row
  // Rows that a workgroup's waves copy at once, and how often they do a step.
  constexpr int rows_at_once(int hd, int waves) { return 64 * waves / pieces(hd); }
  constexpr int copies(int hd, int waves, int keys) { return keys / rows_at_once(hd, waves); }

  // Where a lane's first read lies, and those of the copies after it.
  constexpr unsigned lane_at(int row, int piece, unsigned step) { return row * step + 16u * piece; }
  constexpr unsigned copy_at(unsigned lane, int copy, int at_once, unsigned step)
  {
    return lane + static_cast<unsigned>(copy * at_once) * step;
  }

  // The bytes of `more` rows and one more of `width` halves, `step` bytes apart.
  constexpr unsigned rows_bytes(int more, unsigned step, int width)
  {
    const unsigned long long bytes = static_cast<unsigned long long>(more) * step + 2u * width;
    return bytes < 0xFFFFFFFFull ? static_cast<unsigned>(bytes) : 0xFFFFFFFFu;
  }
} // namespace mi::packed_copies
