// Branches of so many tokens (csrc/page_book.h): all of a sequence's for -1 alone.
#include <cstdio>

#include "../../fyusenet_amd/csrc/page_book.h"

int main() {
    for (int tokens : {-1, 0, 5, 11, -2, -100, -2147483647 - 1, 12, 2147483647}) {
        fynhip::PageBook book(8, 3, 8, 64);
        const int zero[] = {0}, one[] = {1}, counts[] = {11};
        book.extend(1, zero, counts);
        bool refused = false;
        try {
            book.fork(0, 1, one, tokens);
        } catch (const fynhip::PageBook::Refused&) {
            refused = true;
        }
        const bool good = tokens >= -1 && tokens <= 11;
        if (refused == good || book.length(1) != (!good ? 0 : tokens < 0 ? 11 : tokens)) {
            fprintf(stderr, "%d tokens: refused %d, the branch has %d\n", tokens, refused, book.length(1));
            return 1;
        }
    }
    return 0;
}
