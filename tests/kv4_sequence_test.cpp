// The rows and positions of a sequence for whatever the device arrays may hold (ml-drift_amd/csrc/kv4.h), on the host.
#include <climits>
#include <cstdio>

#include "../ml-drift_amd/csrc/kv4.h"

using mldhip::Kv4SequenceFrom;

int main() {
  const int values[] = {INT_MIN, INT_MIN + 1, INT_MIN + 5, -(1 << 30), -7, -1, 0, 1, 5, 59, 60, 61, 1 << 24, (1 << 24) + 1, 1 << 30, INT_MAX - 5, INT_MAX - 1, INT_MAX};
  const int tokens_of[] = {1, 60, 1 << 24}, pages_of[] = {1, 4, 1 << 20}, shift_of[] = {4, 10};
  int bad = 0;
  auto within = [](long long v, long long low, long long high) { return v < low ? low : v > high ? high : v; };
  for (int tokens : tokens_of)
    for (int pages : pages_of)
      for (int shift : shift_of)
        for (int from : values)
          for (int to : values)
            for (int length : values) {
              const mldhip::Kv4Sequence q = Kv4SequenceFrom(from, to, length, tokens, pages, shift);
              const long long start = within(from, 0, tokens), end = within(to, 0, tokens), count = end > start ? end - start : 0;
              const long long held = within(length, 0, 1 << 30), room = (long long)pages << shift;
              if (q.start != start || q.count != count || q.first != held - count || q.held != (held < room ? held : room)) {
                if (bad++ < 5)
                  std::printf("from %d to %d length %d of %d rows, %d pages of 2^%d: start %d count %d first %d held %d\n", from, to, length, tokens, pages, shift,
                              q.start, q.count, q.first, q.held);
              }
            }
  if (bad) return std::printf("%d bad\n", bad), 1;
  std::printf("sequences ok\n");
  return 0;
}
