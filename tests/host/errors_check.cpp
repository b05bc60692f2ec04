// Prints what an engine reports for each pair of error words given on stdin: a wait code and the pages' bits.
#include <iostream>

#include "errors.h"

int main() {
    int wait = 0, bits = 0;
    while (std::cin >> wait >> bits) std::cout << laic::step_error_text(wait, bits) << "\n";
    return 0;
}
